// kv_append.hip -- keys and values of new tokens stored in a paged KV cache for gfx950, with the
// position rotation of q and k on the way.
//
// Token t of sequence b has position p = start[b] + t - cu[b].  For i < rotary / 2 the angle is
// p * inv_freq[i], and the pair (x, y) = dims (i, i + rotary / 2), or (2i, 2i + 1) interleaved,
// becomes (x cos - y sin, x sin + y cos); the other dims stay.  k goes to its page rotated, v as it
// is: as bf16, or divided by the head's scale and rounded once to e4m3 (values past +-448 saturate,
// NaN stays).  q and, when asked for, k are also returned rotated, as bf16.
//
// The angle is formed in 64 bits, in turns (p * inv_freq / 2 pi) with its whole turns taken off before
// it is narrowed: at p = 10^6 a float32 angle would be off by 0.03 rad.  sincospi of the rest, the
// rotation and the division are float32, each output rounded once.
//
// Bound: bytes (every vector is read once and written once) for prompts, latency at decode.  One
// workgroup of 256 threads takes up to 16 head vectors of a token at a time, 16 lanes of 8 dims each:
// with halves paired a lane holds dims 4s .. + 3 of both halves, so that a pair never leaves its lane.
// The token's cosines are computed once per workgroup, one per thread, and shared through LDS; the
// first vectors are on their way meanwhile.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"

#include <algorithm>

namespace nmi {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerPass = kThreads / 16;

// 8 dims of a head vector: quads at d0 and d1
struct Dims {
    int d0, d1;
};

__device__ __forceinline__ void load8(const uint16_t* p, Dims d, float (&x)[8]) {
    const uint2 lo = *reinterpret_cast<const uint2*>(p + d.d0), hi = *reinterpret_cast<const uint2*>(p + d.d1);
    x[0] = bf16lo_to_f32(lo.x), x[1] = bf16hi_to_f32(lo.x), x[2] = bf16lo_to_f32(lo.y), x[3] = bf16hi_to_f32(lo.y);
    x[4] = bf16lo_to_f32(hi.x), x[5] = bf16hi_to_f32(hi.x), x[6] = bf16lo_to_f32(hi.y), x[7] = bf16hi_to_f32(hi.y);
}

__device__ __forceinline__ void store8(uint16_t* p, Dims d, const float (&x)[8]) {
    *reinterpret_cast<uint2*>(p + d.d0) = uint2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    *reinterpret_cast<uint2*>(p + d.d1) = uint2{pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

// x / s as an e4m3 code: to the nearest (ties to even), saturating
__device__ __forceinline__ float to_e4m3_range(float x, float s) {
    const float y = x / s;
    return y > 448.f ? 448.f : (y < -448.f ? -448.f : y);      // (NaN stays)
}
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <bool E4M3>
__device__ __forceinline__ void store_cache(uint8_t* p, Dims d, const float (&x)[8], float s) {
    if constexpr (E4M3) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = to_e4m3_range(x[i], s);
        *reinterpret_cast<uint32_t*>(p + d.d0) = pack_e4m3(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint32_t*>(p + d.d1) = pack_e4m3(y[4], y[5], y[6], y[7]);
    } else {
        store8(reinterpret_cast<uint16_t*>(p), d, x);
    }
}

// The sequence of packed row t: the number of ends cu[1 ..] at or before it (64 of them at a time).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int t, int lane) {
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const int i = b0 + lane;
        const bool before = i < batch && cu[i + 1] <= t;
        const int n = __popcll(__builtin_amdgcn_ballot_w64(before));
        if (n < 64) return b0 + n;
    }
    return batch;
}

template <bool E4M3, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const AppendArgs a) {
    __shared__ float2 turn[kPagedHead / 2];         // cos, sin of each frequency
    const int t = blockIdx.x, tid = threadIdx.x;
    int b = t, place = 0;
    if (a.cu) {
        b = __builtin_amdgcn_readfirstlane(sequence_of(a.cu, a.batch, t, tid & 63));
        if (b >= a.batch) return;                   // rows behind the last sequence
        place = t - a.cu[b];
        if (place < 0) return;                      // rows before the first
    }
    const int start = a.start[b];
    if (start < 0) return;                          // a sequence that is not in use
    const int64_t pos = (int64_t)start + place;

    const int sub = tid & 15;
    const int nq = a.q ? a.H : 0, n_kv = a.kv.n_kv, rows = nq + 2 * n_kv;
    const int pairs = a.rotary / 8;                 // lanes of a vector that rotate
    const bool rotates = sub < pairs;
    // the lane's dims in a vector that is rotated, and in one that is not
    const Dims plain{8 * sub, 8 * sub + 4};
    const Dims turned = (rotates && !INTERLEAVED) ? Dims{4 * sub, a.rotary / 2 + 4 * sub} : plain;

    float x[8];
    int row = blockIdx.y * kRowsPerPass + (tid >> 4);
    auto load = [&](int r) {
        if (r < nq) load8(a.q + (int64_t)t * a.ldq + r * kPagedHead, turned, x);
        else if (r < nq + n_kv) load8(a.k + (int64_t)t * a.ldk + (r - nq) * kPagedHead, turned, x);
        else load8(a.v + (int64_t)t * a.ldv + (r - nq - n_kv) * kPagedHead, plain, x);
    };
    if (row < rows) load(row);

    if (a.rotary) {
        if (tid < a.rotary / 2) {
            const double turns = (double)pos * (double)a.inv_freq[tid] * 0.15915494309189535;   // 1 / (2 pi)
            float s, c;
            sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
            turn[tid] = float2{c, s};
        }
        __syncthreads();
    }
    // where the token goes; nowhere if the table has no page for it
    uint8_t *kp = nullptr, *vp = nullptr;
    {
        bool bad = false;
        const int64_t entry = pos >> a.kv.page_shift;
        int page = 0;
        if (entry < a.kv.max_pages) page = checked_page(a.kv.page_table[b * a.kv.table_stride + entry], a.kv.n_pages, &bad);
        else bad = true;
        if (!bad) {
            const int64_t off = page * a.kv.page_stride + (pos & ((1 << a.kv.page_shift) - 1)) * a.kv.token_stride;
            kp = a.kv.k_pages + off;
            vp = a.kv.v_pages + off;
        } else if (tid == 0 && a.kv.error) {
            __hip_atomic_store(a.kv.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
    while (row < rows) {
        if (row < nq + n_kv) {
            if (rotates) {
                float c[4], s[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 cs = turn[4 * sub + i];
                    c[i] = cs.x, s[i] = cs.y;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    constexpr int second = INTERLEAVED ? 1 : 4;
                    const int i0 = INTERLEAVED ? 2 * i : i;
                    const float u = x[i0], w = x[i0 + second];
                    x[i0] = u * c[i] - w * s[i];
                    x[i0 + second] = u * s[i] + w * c[i];
                }
            }
            if (row < nq) {
                store8(a.q_out + (int64_t)t * a.ldqo + row * kPagedHead, turned, x);
            } else {
                const int h = row - nq;
                if (a.k_out) store8(a.k_out + (int64_t)t * a.ldko + h * kPagedHead, turned, x);
                if (kp)
                    store_cache<E4M3>(kp + h * a.kv.head_stride, turned, x, E4M3 && a.kv.k_scale ? a.kv.k_scale[h] : 1.f);
            }
        } else if (vp) {
            const int h = row - nq - n_kv;
            store_cache<E4M3>(vp + h * a.kv.head_stride, plain, x, E4M3 && a.kv.v_scale ? a.kv.v_scale[h] : 1.f);
        }
        row += kRowsPerPass * gridDim.y;
        if (row < rows) load(row);
    }
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs& a, bool e4m3, hipStream_t stream) {
    const int rows = (a.q ? a.H : 0) + 2 * a.kv.n_kv;
    const int passes = (rows + kRowsPerPass - 1) / kRowsPerPass;
    const dim3 grid(a.tokens, passes);
    if (e4m3) {
        if (a.interleaved) hipLaunchKernelGGL((kv_append_kernel<true, true>), grid, dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((kv_append_kernel<true, false>), grid, dim3(kThreads), 0, stream, a);
    } else {
        if (a.interleaved) hipLaunchKernelGGL((kv_append_kernel<false, true>), grid, dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((kv_append_kernel<false, false>), grid, dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace nmi
