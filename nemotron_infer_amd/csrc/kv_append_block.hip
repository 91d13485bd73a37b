// kv_append_block.hip -- keys and values of new tokens stored as e4m3 in a paged KV cache under a scale for
// each head and block of 16 positions, for gfx950, with the position rotation of q and k on the way.
//
// Positions, rotation and outputs are kv_append.hip's.  A block's scale is a power of two: the smallest s with
// |x| <= 448 s for the new tokens' finite values, no less than the block's scale so far where it held
// positions before (a block whose first place is new begins anew).  Codes are rne(x / s); where s grew, the
// block's earlier codes become rne(code s_old / s).  Powers of two, so that a block filled a token at a time
// is as good as one filled at once: a code that moves to a larger scale loses bits only where it becomes
// subnormal (below 2^-15 of the block's largest value), and x / s is exact before its one rounding.
//
// The largest value decides a scale, so k is rotated in 64 bits and rounded to float32 once (each product of
// a bf16 and a float32 is exact there): equal inputs give equal scales however the rotation is computed.
// NaN and infinities become NaN (e4m3 has no infinity) and do not count for the scale.
//
// Bound: bytes for prompts, latency at decode.  Prompts: a workgroup takes a block of a sequence's positions, or a part of
// its heads, and forms the cosines of its 16 tokens once, in LDS; a wave takes a head's 16 vectors at a time, 8 lanes to
// each, so that their largest value is a matter of its own lanes, and the block's earlier codes are at hand to move.  Decode:
// a wave takes the token or some of its vectors, as in kv_append.hip, and each 8 lanes see to their vector's block.
// Measured: 8191 tokens of 40 / 8 heads 51.2 us (4.6 TB/s read and written; a large copy: 4.9), 42.8 with outputs that stay in
// the last-level cache; one token of 24 sequences 3.3 (graph replays).  With the first loads ahead of the look-up of
// their place, or the next head's ahead of this one's stores, 46.4 and 44.6 where it takes 42.8.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

#include <algorithm>

namespace nmi {

namespace {

constexpr int kWaves = 4;
// Times 8 query vectors of a wave on their way at once.  1 / 2 / 4 (inputs and outputs past the last-level cache, rotated, 40 / 8
// heads): 8191 tokens 51.7 / 51.7 / 51.2 us, 8 prompts of 1000 50.7 / 50.4 / 50.0, 5 of up to 1801 24.4 / 23.7 / 23.5.
constexpr int kAhead = 4;
enum { kPlain = 0, kHalves = 1, kInterleaved = 2 };

// The largest of m and the finite values' magnitudes, as bits.
__device__ __forceinline__ uint32_t finite_max(const float (&x)[8], uint32_t m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        m = b < 0x7F800000u ? max(m, b) : m;
    }
    return m;
}
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    const int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// Codes of x / s, inv = 1 / s; what is not finite is NaN.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fabsf(x[i]) < INFINITY ? x[i] * inv : NAN;
    return uint2{pack4_e4m3(y[0], y[1], y[2], y[3]), pack4_e4m3(y[4], y[5], y[6], y[7])};
}
// Codes times f <= 1.
__device__ __forceinline__ uint32_t codes4_times(uint32_t w, float f) {
    const uint2 b = e4m3x4_to_bf16(w);
    return pack4_e4m3(bf16lo_to_f32(b.x) * f, bf16hi_to_f32(b.x) * f, bf16lo_to_f32(b.y) * f, bf16hi_to_f32(b.y) * f);
}
__device__ __forceinline__ uint4 codes16_times(uint4 w, float f) {
    return uint4{codes4_times(w.x, f), codes4_times(w.y, f), codes4_times(w.z, f), codes4_times(w.w, f)};
}

// A block's new scale and what goes with it.
struct Scale {
    float s, inv, moved;        // moved: s_old / s, of the earlier codes; 1 where they stay
};
__device__ __forceinline__ Scale new_scale(uint32_t amax, bool had, uint32_t old_bits) {
    int e = block_exponent(amax);
    if (had) e = max(e, block_exponent_of_scale(old_bits));
    Scale n;
    n.s = __uint_as_float((uint32_t)e << 23);
    n.inv = __uint_as_float((uint32_t)(254 - e) << 23);
    n.moved = had ? __uint_as_float(old_bits) * n.inv : 1.f;
    return n;
}

// a ca + b cb, to the nearest float32: both products are exact in 64 bits (8 by 24).
__device__ __forceinline__ float turned(float a, float ca, float b, float cb) {
    return (float)__builtin_fma((double)a, (double)ca, (double)b * (double)cb);
}
template <bool EXACT>
__device__ __forceinline__ void rotate_pair(float& x, float& y, float c, float s) {
    const float u = x, w = y;
    if constexpr (EXACT) {
        x = turned(u, c, -w, s);
        y = turned(u, s, w, c);
    } else {
        x = __builtin_fmaf(u, c, -(w * s));
        y = __builtin_fmaf(u, s, w * c);
    }
}
// The lane's two times 8 dims of a vector: those of both halves of the same pairs, or 16 neighbours.
template <int MODE, bool EXACT>
__device__ __forceinline__ void rotate(float (&x)[8], float (&y)[8], const float2* turns, bool turns_here) {
    if (MODE == kPlain || !turns_here) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 t = turns[j];
        if constexpr (MODE == kHalves) {
            rotate_pair<EXACT>(x[j], y[j], t.x, t.y);
        } else {
            float(&z)[8] = j < 4 ? x : y;
            const int e = 2 * (j & 3);
            rotate_pair<EXACT>(z[e], z[e + 1], t.x, t.y);
        }
    }
}

// What a lane (sub: its place among the vector's 8) takes of a vector.
template <int MODE>
struct Dims {
    int p0, r0, r1;             // not rotated: p0 .. + 15; rotated: r0 .. + 7 and r1 .. + 7
    bool turns;                 // these are rotated
    __device__ Dims(int sub, int rotary) {
        p0 = 16 * sub;
        const bool halves = MODE == kHalves && sub < rotary / 16;
        r0 = halves ? 8 * sub : p0;
        r1 = halves ? rotary / 2 + 8 * sub : p0 + 8;
        turns = MODE == kHalves ? halves : p0 < rotary;
    }
};

__device__ __forceinline__ void angles(const AppendArgs& a, int64_t pos, int i, float2* t) {
    const double turn = (double)pos * (double)a.inv_freq[i] * 0.15915494309189535;       // 1 / (2 pi)
    cos_sin(turn - rint(turn), &t->x, &t->y);
}

// Where position pos of sequence b goes: the byte offset in the pools and the index of head 0's scale; false, and
// reported by the lane that is told to, where the table has no page for it.
struct Where {
    int64_t off, block;         // block: of head h, + h << (page_shift - 4)
};
__device__ __forceinline__ bool find_place(const PagedKv& kv, int b, int64_t pos, bool tell, Where* w) {
    bool bad = false;
    const int64_t entry = pos >> kv.page_shift;
    int page = 0;
    if (entry < kv.max_pages) page = checked_page(load_const(kv.page_table + b * kv.table_stride + entry), kv.n_pages, &bad);
    else bad = true;
    if (bad) {
        if (tell) report(kv.error);
        return false;
    }
    const int in_page = (int)(pos & ((1 << kv.page_shift) - 1));
    w->off = page * kv.page_stride + in_page * kv.token_stride;
    w->block = block_index(page, kv.n_kv, 0, kv.page_shift, in_page);
    return true;
}

// One new token per sequence: a wave takes the token or a part of its head vectors, 8 at a time, 8 lanes each.
template <int MODE>
__global__ __launch_bounds__(64 * kWaves) void kv_append_block_token_kernel(const AppendArgs a, int parts) {
    __shared__ float2 turns[kWaves][kPagedHead / 2];
    const int tid = threadIdx.x, lane = tid & 63, sub = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t job = (int64_t)blockIdx.x * kWaves + wave;
    const int t = (int)(job / parts), part = (int)(job - (int64_t)t * parts);
    if (t >= a.tokens) return;
    const Dims<MODE> d(sub, a.rotary);
    const int nq = a.q ? a.H : 0, n_kv = a.kv.n_kv, rows = nq + 2 * n_kv;
    uint4 lo, hi;
    auto load = [&](int pass) {
        const int row = 8 * pass + (lane >> 3);
        if (row < rows) {
            const bool is_q = row < nq, is_v = row >= nq + n_kv;
            const uint16_t* x = is_q   ? a.q + (int64_t)t * a.ldq + row * kPagedHead
                                : is_v ? a.v + (int64_t)t * a.ldv + (row - nq - n_kv) * kPagedHead
                                       : a.k + (int64_t)t * a.ldk + (row - nq) * kPagedHead;
            lo = load16(x + (is_v ? d.p0 : d.r0));
            hi = load16(x + (is_v ? d.p0 + 8 : d.r1));
        }
    };
    load(part);
    const int start = load_const(a.start + t);
    if (start < 0) return;
    Where at;
    const bool stored = find_place(a.kv, t, start, lane == 0, &at);
    const int before = start & (kPagedBlock - 1);               // places of the block that were filled earlier
    if constexpr (MODE != kPlain) {
        if (lane < a.rotary / 2) angles(a, start, lane, &turns[wave][lane]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (a wave's own: no barrier)
        __builtin_amdgcn_wave_barrier();
    }
    const int passes = (rows + 7) / 8;
    for (int pass = part; pass < passes; pass += parts) {
        if (pass != part) load(pass);
        const int row = 8 * pass + (lane >> 3);
        if (row >= rows) continue;
        const bool is_q = row < nq, is_v = row >= nq + n_kv;
        float x[8], y[8];
        unpack8(lo, x);
        unpack8(hi, y);
        if (MODE != kPlain && is_q) {
            rotate<MODE, false>(x, y, &turns[wave][8 * sub], d.turns);
            uint16_t* o = a.q_out + (int64_t)t * a.ldqo + row * kPagedHead;
            *reinterpret_cast<uint4*>(o + d.r0) = pack8(x);
            *reinterpret_cast<uint4*>(o + d.r1) = pack8(y);
            continue;
        }
        const int h = is_v ? row - nq - n_kv : row - nq;
        if (!is_v) rotate<MODE, true>(x, y, &turns[wave][8 * sub], d.turns);
        const int d0 = is_v ? d.p0 : d.r0, d1 = is_v ? d.p0 + 8 : d.r1;
        if (MODE != kPlain && !is_v && a.k_out) {
            uint16_t* o = a.k_out + (int64_t)t * a.ldko + h * kPagedHead;
            *reinterpret_cast<uint4*>(o + d0) = pack8(x);
            *reinterpret_cast<uint4*>(o + d1) = pack8(y);
        }
        if (!stored) continue;
        uint8_t* p = (is_v ? a.kv.v_pages : a.kv.k_pages) + at.off + h * a.kv.head_stride;
        float* sp = (is_v ? a.blocks.v : a.blocks.k) + at.block + ((int64_t)h << (a.kv.page_shift - 4));
        const uint32_t old = before ? __float_as_uint(*sp) : 0u;
        uint32_t m = finite_max(y, finite_max(x, 0u));          // over the vector's 8 lanes
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
        const Scale n = new_scale(m, before > 0, old);
        *reinterpret_cast<uint2*>(p + d0) = codes8(x, n.inv);
        *reinterpret_cast<uint2*>(p + d1) = codes8(y, n.inv);
        if (!before || n.moved != 1.f) {
            if (sub == 0) *sp = n.s;
            // the block's earlier codes: a row by the 8 lanes, 8 rows on their way at once
#pragma unroll
            for (int r0 = 1; r0 < kPagedBlock; r0 += 8) {
                if (r0 > before) break;
                uint4 w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (r0 + i <= before) w[i] = load16(p - (r0 + i) * a.kv.token_stride + 16 * sub);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (r0 + i <= before)
                        *reinterpret_cast<uint4*>(p - (r0 + i) * a.kv.token_stride + 16 * sub) = codes16_times(w[i], n.moved);
            }
        }
    }
}

// Packed rows: a workgroup's job is a block of positions of a sequence that new tokens lie in.
struct Job {
    int b, row, n;              // sequence; its first new token's row, and how many new ones the block has
    int64_t pos;                // the first one's position
};
__device__ __forceinline__ bool find_job(const AppendArgs& a, uint32_t x, int lane, Job* job) {
    Packed s;
    if (!find_packed(a.cu, a.start, a.batch, a.tokens, x, lane, [](int64_t pos, int rows) { return blocks_of(pos, rows); }, &s))
        return false;
    const int64_t block = s.pos / kPagedBlock + s.k;
    const int64_t begin = s.k ? block * kPagedBlock : s.pos, stop = std::min((block + 1) * kPagedBlock, s.pos + s.rows);
    *job = Job{s.b, s.row + (int)(begin - s.pos), (int)(stop - begin), begin};
    return true;
}

template <int MODE>
__global__ __launch_bounds__(64 * kWaves) void kv_append_block_kernel(const AppendArgs a) {
    __shared__ float2 turns[kPagedBlock][kPagedHead / 2];       // cos, sin of each token's frequencies
    const int tid = threadIdx.x, lane = tid & 63, sub = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = blockIdx.y, parts = gridDim.y;
    if (blockIdx.x + 1 == gridDim.x) {
        if (part == 0 && wave == 0) check_offsets(a.cu, a.batch, a.tokens, a.kv.error, lane);
        return;
    }
    Job job;
    if (!find_job(a, blockIdx.x, lane, &job)) return;
    Where at;
    const bool stored = find_place(a.kv, job.b, job.pos, part == 0 && tid == 0, &at);
    const int before = (int)(job.pos & (kPagedBlock - 1));
    if constexpr (MODE != kPlain) {
        const int half = a.rotary / 2;
        for (int i = tid; i < job.n * half; i += 64 * kWaves) angles(a, job.pos + i / half, i % half, &turns[i / half][i % half]);
        __syncthreads();
    }
    const Dims<MODE> d(sub, a.rotary);
    const int n_kv = a.kv.n_kv;
    // a wave takes a KV head's keys or values of all the block's new tokens
    for (int task = part * kWaves + wave; task < 2 * n_kv; task += parts * kWaves) {
        const bool is_v = task >= n_kv;
        const int h = is_v ? task - n_kv : task;
        const uint16_t* src = (is_v ? a.v + job.row * a.ldv : a.k + job.row * a.ldk) + h * kPagedHead;
        const int64_t ld = is_v ? a.ldv : a.ldk;
        const int d0 = is_v ? d.p0 : d.r0, d1 = is_v ? d.p0 + 8 : d.r1;
        uint4 lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tok = (lane >> 3) + 8 * i;
            lo[i] = hi[i] = uint4{0, 0, 0, 0};
            if (tok < job.n) {
                lo[i] = load16(src + tok * ld + d0);
                hi[i] = load16(src + tok * ld + d1);
            }
        }
        uint8_t* p = (is_v ? a.kv.v_pages : a.kv.k_pages) + at.off + h * a.kv.head_stride;
        float* sp = (is_v ? a.blocks.v : a.blocks.k) + at.block + ((int64_t)h << (a.kv.page_shift - 4));
        const uint32_t old = stored && before ? __float_as_uint(*sp) : 0u;
        float x[2][8], y[2][8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tok = (lane >> 3) + 8 * i;
            unpack8(lo[i], x[i]);
            unpack8(hi[i], y[i]);
            if (tok < job.n) {
                if (!is_v) {
                    rotate<MODE, true>(x[i], y[i], &turns[tok][8 * sub], d.turns);
                    if (MODE != kPlain && a.k_out) {
                        uint16_t* o = a.k_out + (int64_t)(job.row + tok) * a.ldko + h * kPagedHead;
                        *reinterpret_cast<uint4*>(o + d0) = pack8(x[i]);
                        *reinterpret_cast<uint4*>(o + d1) = pack8(y[i]);
                    }
                }
                m = finite_max(y[i], finite_max(x[i], m));
            }
        }
        if (!stored) continue;
        const Scale n = new_scale(wave_max_u32(m), before > 0, old);
        if (lane == 0) *sp = n.s;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tok = (lane >> 3) + 8 * i;
            if (tok < job.n) {
                *reinterpret_cast<uint2*>(p + tok * a.kv.token_stride + d0) = codes8(x[i], n.inv);
                *reinterpret_cast<uint2*>(p + tok * a.kv.token_stride + d1) = codes8(y[i], n.inv);
            }
        }
        if (n.moved != 1.f) {                                   // the block's earlier codes
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 1 + (lane >> 3) + 8 * i;          // rows before the first new one
                if (r <= before) {
                    uint4* q = reinterpret_cast<uint4*>(p - r * a.kv.token_stride + 16 * sub);
                    *q = codes16_times(*q, n.moved);
                }
            }
        }
    }
    if (MODE == kPlain || !a.q) return;
    // q: 8 vectors at a time, the heads of a token one after another, kAhead times that on their way at once
    const int vectors = job.n * a.H, stride = 8 * parts * kWaves;
    for (int v0 = 8 * (part * kWaves + wave) + (lane >> 3); __builtin_amdgcn_ballot_w64(v0 < vectors); v0 += kAhead * stride) {
        uint4 lo[kAhead], hi[kAhead];
        int tok[kAhead], h[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int v = v0 + i * stride;
            tok[i] = v / a.H;
            h[i] = v - tok[i] * a.H;
            if (v < vectors) {
                const uint16_t* src = a.q + (int64_t)(job.row + tok[i]) * a.ldq + h[i] * kPagedHead;
                lo[i] = load16(src + d.r0);
                hi[i] = load16(src + d.r1);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (v0 + i * stride >= vectors) break;
            float x[8], y[8];
            unpack8(lo[i], x);
            unpack8(hi[i], y);
            rotate<MODE, false>(x, y, &turns[tok[i]][8 * sub], d.turns);
            uint16_t* o = a.q_out + (int64_t)(job.row + tok[i]) * a.ldqo + h[i] * kPagedHead;
            *reinterpret_cast<uint4*>(o + d.r0) = pack8(x);
            *reinterpret_cast<uint4*>(o + d.r1) = pack8(y);
        }
    }
}

template <int MODE>
void launch(const AppendArgs& a, hipStream_t stream) {
    const int vectors = (a.q ? a.H : 0) + 2 * a.kv.n_kv, cus = device_info().num_cu;
    if (!a.cu) {
        const int passes = (vectors + 7) / 8;
        const int parts = std::min(passes, std::max(1, 8 * cus / a.tokens));
        const int64_t jobs = (int64_t)a.tokens * parts;
        hipLaunchKernelGGL((kv_append_block_token_kernel<MODE>), dim3((uint32_t)((jobs + kWaves - 1) / kWaves)),
                           dim3(64 * kWaves), 0, stream, a, parts);
        return;
    }
    // A block's heads in as many parts as leave four workgroups to a CU (2 / 4 / 8 of them: 8191 tokens 51.5 / 51.2 / 52.5 us,
    // 5 prompts of up to 1801 24.3 / 23.5 / 23.5, of 16 / 4 heads 10.8 / 11.1 / 12.5).
    const int64_t jobs = most_blocks(a.tokens, a.batch);
    const int most = (vectors + kWaves - 1) / kWaves;
    const int parts = (int)std::min<int64_t>(most, std::max<int64_t>(1, 4 * cus / jobs));
    hipLaunchKernelGGL((kv_append_block_kernel<MODE>), dim3((uint32_t)jobs + 1, parts), dim3(64 * kWaves), 0, stream, a);
}

}  // namespace

hipError_t launch_kv_append_block(const AppendArgs& a, hipStream_t stream) {
    if (!a.rotary) launch<kPlain>(a, stream);
    else if (!a.interleaved) launch<kHalves>(a, stream);
    else launch<kInterleaved>(a, stream);
    return hipGetLastError();
}

}  // namespace nmi
