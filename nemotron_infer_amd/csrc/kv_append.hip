// kv_append.hip -- keys and values of new tokens stored in a paged KV cache for gfx950, with the
// position rotation of q and k on the way.
//
// Token t of sequence b has position p = start[b] + t - cu[b].  For i < rotary / 2 the angle is
// p * inv_freq[i], and the pair (x, y) = dims (i, i + rotary / 2), or (2i, 2i + 1) interleaved,
// becomes (x cos - y sin, x sin + y cos); the other dims stay.  k goes to its page rotated, v as it
// is: as bf16, or divided by the head's scale and rounded once to e4m3 (values past +-448 saturate,
// NaN stays).  q and, when asked for, k are also returned rotated, as bf16.
//
// The angle is formed in 64 bits, in turns (p * inv_freq / 2 pi) with its whole turns taken off (at
// p = 10^6 a float32 angle would be off by 0.03 rad), and so are its sine and cosine (cos_sin), each
// rounded once; the rotation and the division are float32, each output rounded once.
//
// Bound: bytes (every vector is read once and written once) for prompts, latency at decode.  A wave
// takes a token, or a part of its head vectors where there are few tokens: 8 vectors at a time, 8 lanes
// of two times 8 dims each, BATCH times that on their way at once.  With halves paired a lane
// holds the same 8 dims of both halves, so that a pair never leaves its lane.  The token's cosines are
// computed once per wave, one per lane, while the vectors are on their way, and passed on through LDS.
// Measured (40 / 8 heads, rotated; graph replays): one token 3.0-3.7 us, 8191 tokens into an e4m3 cache 48
// us, 4.9 TB/s read and written (a large copy: 4.9); with a workgroup to a token, 8-byte rows and a
// float32 sine, 71 us.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"

#include <algorithm>

namespace nmi {

namespace {

constexpr int kWaves = 4;
// Times 8 vectors that a wave that takes several asks for at once: few registers and so more waves, which hide
// more than longer batches do.  2 / 4 / 7 (graph replays, rotated): 8191 tokens of 40 / 8 heads into bf16
// 51.0 / 50.9 / 54.6 us, into e4m3 48.2 / 48.8 / 52.1, of 32 / 8 44.4 / 45.4 / 49.1, of 16 / 4 24.8 / 25.8 / 25.9, 64
// interleaved dims 59.3 / 59.9 / 59.4; k and v alone 14.3 / 14.2 / 15.0; 600 tokens 6.5 / 6.75 / 6.8.
constexpr int kBatch = 2;
enum { kPlain = 0, kHalves = 1, kInterleaved = 2 };

__device__ __forceinline__ void unpack8(const uint4 v, float (&x)[8]) {
    const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = bf16lo_to_f32(d[i]), x[2 * i + 1] = bf16hi_to_f32(d[i]);
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return uint4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

// x / s as an e4m3 code: to the nearest (ties to even), saturating; NaN stays
__device__ __forceinline__ float to_e4m3_range(float x, float s) {
    const float y = x / s;
    return y > 448.f ? 448.f : (y < -448.f ? -448.f : y);
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&x)[8], float s) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_e4m3_range(x[i], s);
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), b = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], b, true);
    return uint2{(uint32_t)a, (uint32_t)b};
}

// The sequence of packed row t and t's place in it, 64 sequences at a time: the first of several that have the
// row (offsets that fall), -1 where none has.
__device__ __forceinline__ int find_sequence(const AppendArgs& a, int t, int lane, int* place) {
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int i = b0 + lane;
        int c0 = 0;
        bool mine = false;
        if (i < a.batch) {
            c0 = a.cu[i];
            mine = span_holds(c0, a.cu[i + 1], t);
        }
        if (const uint64_t holds = __builtin_amdgcn_ballot_w64(mine)) {
            const int who = __builtin_ctzll(holds);
            *place = span_place(__builtin_amdgcn_readlane(c0, who), t);
            return b0 + who;
        }
    }
    return -1;
}
// Reports offsets out of order or range.  The work of a wave of its own, behind those of the tokens: in theirs
// the checks cost 150 to 600 tokens 0.2 us of 4 to 7.
__device__ __forceinline__ void check_offsets(const AppendArgs& a, int lane) {
    bool bad = false;
    for (int i = lane; i < a.batch; i += 64) {
        int first;
        checked_span(a.cu[i], a.cu[i + 1], a.tokens, &first, &bad);
    }
    if (bad && a.kv.error) __hip_atomic_store(a.kv.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// parts: waves that share a token, BATCH its vectors (by 8) on their way at once.
template <bool E4M3, int MODE, int BATCH>
__global__ __launch_bounds__(64 * kWaves) void kv_append_kernel(const AppendArgs a, int parts) {
    __shared__ float2 turns[kWaves][kPagedHead / 2];            // cos, sin of each frequency
    const int tid = threadIdx.x, lane = tid & 63, sub = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t job = (int64_t)blockIdx.x * kWaves + wave;
    const int t = (int)(job / parts), part = (int)(job - (int64_t)t * parts);
    if (t >= a.tokens) {
        if (a.cu && t == a.tokens && part == 0) check_offsets(a, lane);
        return;
    }

    // the lane's two times 8 dims in a vector that is rotated, and in one that is not
    const int turning = a.rotary / 16;                          // lanes of a vector that rotate (halves)
    const int p0 = 16 * sub, p1 = p0 + 8;
    const bool halves = MODE == kHalves && sub < turning;
    const int r0 = halves ? 8 * sub : p0, r1 = halves ? a.rotary / 2 + 8 * sub : p1;

    const int nq = a.q ? a.H : 0, n_kv = a.kv.n_kv, rows = nq + 2 * n_kv;
    uint4 lo[BATCH], hi[BATCH];
    auto load = [&](int pass0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int row = 8 * (pass0 + i * parts) + (lane >> 3);
            if (row < rows) {
                const bool is_q = row < nq, is_v = row >= nq + n_kv;
                const uint16_t* x = is_q   ? a.q + (int64_t)t * a.ldq + row * kPagedHead
                                    : is_v ? a.v + (int64_t)t * a.ldv + (row - nq - n_kv) * kPagedHead
                                           : a.k + (int64_t)t * a.ldk + (row - nq) * kPagedHead;
                lo[i] = load16(x + (is_v ? p0 : r0));
                hi[i] = load16(x + (is_v ? p1 : r1));
            }
        }
    };
    load(part);

    int b = t, place = 0;
    if (a.cu) {
        b = find_sequence(a, t, lane, &place);
        if (b < 0) return;                                      // rows of no sequence
    }
    const int start = load_const(a.start + b);
    if (start < 0) return;                                      // a sequence that is not in use
    const int64_t pos = (int64_t)start + place;

    // where the token goes; nowhere if the table has no page for it
    uint8_t *kp = nullptr, *vp = nullptr;
    {
        bool bad = false;
        const int64_t entry = pos >> a.kv.page_shift;
        int page = 0;
        if (entry < a.kv.max_pages)
            page = checked_page(load_const(a.kv.page_table + b * a.kv.table_stride + entry), a.kv.n_pages, &bad);
        else
            bad = true;
        if (!bad) {
            const int64_t off = page * a.kv.page_stride + (pos & ((1 << a.kv.page_shift) - 1)) * a.kv.token_stride;
            kp = a.kv.k_pages + off;
            vp = a.kv.v_pages + off;
        } else if (lane == 0 && a.kv.error) {
            __hip_atomic_store(a.kv.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
    float c[8], s[8];                                           // of the lane's pairs
    if constexpr (MODE != kPlain) {
        if (lane < a.rotary / 2) {
            const double turn = (double)pos * (double)a.inv_freq[lane] * 0.15915494309189535;   // 1 / (2 pi)
            cos_sin(turn - rint(turn), &turns[wave][lane].x, &turns[wave][lane].y);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (a wave's own: no barrier)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 cs = turns[wave][8 * sub + i];         // (of frequencies past the last: not used)
            c[i] = cs.x, s[i] = cs.y;
        }
    }

    const int passes = (rows + 7) / 8;
    for (int pass0 = part;; load(pass0)) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int row = 8 * (pass0 + i * parts) + (lane >> 3);
            if (row >= rows) continue;
            const bool is_q = row < nq, is_v = row >= nq + n_kv;
            float x[8], y[8];
            unpack8(lo[i], x);
            unpack8(hi[i], y);
            if (!is_v) {
                if constexpr (MODE == kHalves) {
                    if (halves) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float u = x[j], w = y[j];
                            x[j] = __builtin_fmaf(u, c[j], -(w * s[j]));
                            y[j] = __builtin_fmaf(u, s[j], w * c[j]);
                        }
                    }
                } else if constexpr (MODE == kInterleaved) {
                    if (p0 < a.rotary) {                        // (rotary a multiple of 16: both times 8 dims, or none)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float(&z)[8] = j < 4 ? x : y;       // (j is known here: no choice is left)
                            const int e = 2 * (j & 3);
                            const float u = z[e], w = z[e + 1];
                            z[e] = __builtin_fmaf(u, c[j], -(w * s[j]));
                            z[e + 1] = __builtin_fmaf(u, s[j], w * c[j]);
                        }
                    }
                }
            }
            const uint4 xb = pack8(x), yb = pack8(y);
            if (MODE != kPlain && is_q) {
                uint16_t* o = a.q_out + (int64_t)t * a.ldqo + row * kPagedHead;
                *reinterpret_cast<uint4*>(o + r0) = xb;
                *reinterpret_cast<uint4*>(o + r1) = yb;
                continue;
            }
            const int h = is_v ? row - nq - n_kv : row - nq;
            const int d0 = is_v ? p0 : r0, d1 = is_v ? p1 : r1;
            if (MODE != kPlain && !is_v && a.k_out) {
                uint16_t* o = a.k_out + (int64_t)t * a.ldko + h * kPagedHead;
                *reinterpret_cast<uint4*>(o + d0) = xb;
                *reinterpret_cast<uint4*>(o + d1) = yb;
            }
            uint8_t* p = is_v ? vp : kp;
            if (!p) continue;
            p += h * a.kv.head_stride;
            if constexpr (E4M3) {
                const float* scale = is_v ? a.kv.v_scale : a.kv.k_scale;
                const float sc = scale ? scale[h] : 1.f;
                *reinterpret_cast<uint2*>(p + d0) = pack8_e4m3(x, sc);
                *reinterpret_cast<uint2*>(p + d1) = pack8_e4m3(y, sc);
            } else {
                *reinterpret_cast<uint4*>(p + 2 * d0) = xb;
                *reinterpret_cast<uint4*>(p + 2 * d1) = yb;
            }
        }
        pass0 += BATCH * parts;
        if (pass0 >= passes) break;
    }
}

template <bool E4M3, int BATCH>
void launch(const AppendArgs& a, int parts, hipStream_t stream) {
    const int64_t jobs = (int64_t)a.tokens * parts + (a.cu ? 1 : 0);         // and the offsets' check
    const dim3 grid((uint32_t)((jobs + kWaves - 1) / kWaves)), block(64 * kWaves);
    if (!a.rotary) hipLaunchKernelGGL((kv_append_kernel<E4M3, kPlain, BATCH>), grid, block, 0, stream, a, parts);
    else if (!a.interleaved) hipLaunchKernelGGL((kv_append_kernel<E4M3, kHalves, BATCH>), grid, block, 0, stream, a, parts);
    else hipLaunchKernelGGL((kv_append_kernel<E4M3, kInterleaved, BATCH>), grid, block, 0, stream, a, parts);
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs& a, bool e4m3, hipStream_t stream) {
    // Few tokens: their vectors spread over up to 8 waves per CU, since latency is all there is; many: a
    // wave for a token, whose cosines are then computed once.  Parts 1 / 2 / 4 / 7 (40 / 8 heads, rotated,
    // bf16): 128 tokens 6.0 / 4.7 / 3.9 / 3.6 us, 512 7.7 / 6.2 / 5.9 / 5.7, 1024 9.2 / 8.1 / 9.0 / 9.2,
    // 2048 12.9 / 13.1 / 15.1 / 13.9, 8191 51.0 / 49.7 / 49.1 / 48.2 (into e4m3 47.4 / 46.5 / 48.0 / 51.1).
    const int passes = ((a.q ? a.H : 0) + 2 * a.kv.n_kv + 7) / 8;
    const int parts = std::min(passes, std::max(1, 8 * device_info().num_cu / a.tokens));
    if (parts == passes) {
        if (e4m3) launch<true, 1>(a, parts, stream);
        else launch<false, 1>(a, parts, stream);
    } else {
        if (e4m3) launch<true, kBatch>(a, parts, stream);
        else launch<false, kBatch>(a, parts, stream);
    }
    return hipGetLastError();
}

}  // namespace nmi
