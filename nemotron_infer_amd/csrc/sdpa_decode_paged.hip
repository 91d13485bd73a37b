// sdpa_decode_paged.hip -- attention of one new token per sequence over a paged KV cache, for gfx950.
//
//   o[b, h] = sum_s w_s v_s / sum_s w_s over s < len[b],  w_s = exp(scale q[b, h] . k_s)
//
// k_s, v_s: position s of KV head h / group in sequence b's pages, bf16, or e4m3 times the head's
// scale (k's scale goes into the softmax's, v's into the last division).  A sequence of length 0 gets
// 0.  Float32 throughout: the products are exact bf16 products summed by the matrix cores, the
// softmax weights go into the second product in two bf16 parts (hi = bf16(w), lo = bf16(w - hi), 16
// significant bits), the running maximum, row sum and outputs are float32.
//
// Bound: reading the cache.  Every position is read once per KV head, for all query heads of its
// group (up to 16, the columns of a 16x16 matrix product; larger groups in several passes).
//
// Split: a workgroup of 4 waves takes one KV head over a range of one sequence's positions.  The
// ranges come from the lengths, on the device: their sum over the number of workgroups wanted gives
// the positions per split (split_tiles), each sequence has as many splits as it needs, and
// workgroup x finds its own by a scan over the lengths.  So the grid depends on the batch size only, a
// captured graph stays right and balanced as the sequences grow, and one long sequence among short
// ones is split as far as a batch of equal ones.  Sequences of one split are finished by it; the others
// leave (maximum, row sum, sums) that a second kernel joins in a fixed order.
//
// Wave: stages of 8 KiB (16 positions of bf16, 32 of e4m3) brought into LDS by DMA, two stages per
// wave, so that one is on its way while the other is used; no wave waits for another before the end.
// A tile of 16 positions lies within a page: its address is one scalar.  Per tile:
// * S^T = K . Q^T (positions x heads) by 16x16x32 products: a lane then holds 4 positions of one head.
// * weights in base 2 against a running maximum that is raised only when a score exceeds it by 2^8
//   in weight, so that the sums are rarely rescaled.
// * O^T += V^T . P^T: the 32 places of the product's inner dimension are the tile's 16 positions
//   twice, with the weights' hi and lo parts, so one product does both.  V^T comes from the
//   token-major tile by transposing LDS reads (for e4m3, of pairs of dims, whose bytes are then
//   sorted: the even dims of a block go to one product, the odd ones to the next).
#include "nmi_device.hpp"
#include "nmi_launch.hpp"

#include <algorithm>
#include <cfloat>

namespace nmi {

namespace {

constexpr int kD = kPagedHead;
constexpr int kWaves = 4;
constexpr int kStage = 8192;                    // bytes of K and V per stage
constexpr int kStages = 2;                      // per wave
constexpr int kCols = 16;                       // query heads per workgroup
constexpr int kLds = kWaves * kStages * kStage;
constexpr float kLazy = 8.f;                    // log2 of the largest unnormalised weight

__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Uniform values through the scalar cache, whatever the code around them writes.
template <class T>
__device__ __forceinline__ T load_const(const T* p) {
    return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

__device__ __forceinline__ int tiles_of(const PagedDecodeArgs& a, int b, int* len, bool* bad) {
    *len = b < a.batch ? checked_len(a.lens[b], a.kv.max_pages, a.kv.page_shift, bad) : 0;
    return (*len + kPagedTile - 1) / kPagedTile;
}
__device__ __forceinline__ uint32_t splits_of(int tiles, int chunk) {
    return (uint32_t)max(1, (tiles + chunk - 1) / chunk);
}
// Tiles per split, the same in every wave of the launch.
__device__ __forceinline__ int plan_chunk(const PagedDecodeArgs& a, int unit, int lane) {
    uint32_t total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        int len;
        bool bad = false;
        total += lane_u32(wave_scan_u32((uint32_t)tiles_of(a, b0 + lane, &len, &bad)), 63);
    }
    return split_tiles(total, a.budget, unit);
}

// Split `slot` of all splits: its sequence, that sequence's length and splits, and which of them it is.
struct Slot {
    int b, len, nsplit, split;
    bool bad;
};
__device__ __forceinline__ bool find_slot(const PagedDecodeArgs& a, int slot, int chunk, int lane, Slot* s) {
    uint32_t before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        int len;
        bool bad = false;
        const int tiles = tiles_of(a, b0 + lane, &len, &bad);
        const uint32_t n = b0 + lane < a.batch ? splits_of(tiles, chunk) : 0;
        const uint32_t incl = before + wave_scan_u32(n);
        const int i = __popcll(__builtin_amdgcn_ballot_w64(incl <= (uint32_t)slot));
        if (i < 64) {
            s->b = b0 + i;
            s->len = (int)lane_u32((uint32_t)len, i);
            s->nsplit = (int)lane_u32(n, i);
            s->split = slot - (int)(lane_u32(incl, i) - lane_u32(n, i));
            s->bad = (__builtin_amdgcn_ballot_w64(bad) >> i) & 1;
            return true;
        }
        before = lane_u32(incl, 63);
    }
    return false;
}
// The splits before sequence b's first, and its own.
__device__ __forceinline__ int first_slot(const PagedDecodeArgs& a, int b, int chunk, int lane, int* nsplit) {
    uint32_t before = 0;
    for (int b0 = 0;; b0 += 64) {
        int len;
        bool bad = false;
        const int tiles = tiles_of(a, b0 + lane, &len, &bad);
        const uint32_t n = b0 + lane < a.batch ? splits_of(tiles, chunk) : 0;
        const uint32_t incl = before + wave_scan_u32(n);
        if (b < b0 + 64) {
            *nsplit = (int)lane_u32(n, b - b0);
            return (int)(lane_u32(incl, b - b0) - lane_u32(n, b - b0));
        }
        before = lane_u32(incl, 63);
    }
}

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

template <bool E4M3>
struct Form {
    static constexpr int kTiles = E4M3 ? 2 : 1;         // per stage
    static constexpr int kRow = E4M3 ? kD : 2 * kD;     // bytes of a position
    static constexpr int kTile = kPagedTile * kRow;
    static constexpr int kUnit = kWaves * kTiles;       // tiles that give every wave one stage
};

// LDS tiles: row r of 16-byte chunks, chunk c at c ^ swz(r), so that the reads of 16 rows at one chunk
// (K) or at one 32-byte column (V) spread over the banks.
template <bool E4M3>
__device__ __forceinline__ int k_swz(int r) { return E4M3 ? (r >> 1) & 7 : r & 15; }
template <bool E4M3>
__device__ __forceinline__ int v_swz(int r) { return E4M3 ? 2 * ((r >> 1) & 3) : 2 * (r & 7); }

template <bool E4M3>
__global__ __launch_bounds__(64 * kWaves, 2) void sdpa_decode_paged_kernel(const PagedDecodeArgs a) {
    typedef Form<E4M3> F;
    typedef __attribute__((address_space(3))) void lds_void;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y, r0 = blockIdx.z * kCols, nrow = min(kCols, a.group - r0);

    const int chunk = plan_chunk(a, F::kUnit, lane);
    Slot s;
    if (!find_slot(a, blockIdx.x, chunk, lane, &s)) return;
    bool bad = s.bad;
    const int p0 = s.split * chunk * kPagedTile;                         // first position of the split
    const int p1 = min(s.len, p0 + chunk * kPagedTile);                  // past its last
    const int head0 = kvh * a.group + r0;

    // this lane's head as the B operand: of a bf16 cache, step i holds dims 32 i + 8 g .. + 7; of an
    // e4m3 cache, steps 2 i and 2 i + 1 dims 64 i + 16 g .. + 15 (one 16-byte read of k)
    bf16x8 qf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = E4M3 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
        uint4 v{0, 0, 0, 0};
        if (l16 < nrow) v = load16(a.q + (int64_t)s.b * a.ldq + (int64_t)(head0 + l16) * kD + d);
        qf[i] = __builtin_bit_cast(bf16x8, v);
    }

    // DMA: instruction i brings 1 KiB, rows r = (1024 / kRow) i + lane / (kRow / 16) of a tile
    constexpr int kChunks = F::kRow / 16, kDma = F::kTile / 1024;        // per row; per tile
    const int drow = lane / kChunks, dpos = lane % kChunks;
    auto drow_of = [&](int i) { return drow + (64 / kChunks) * i; };
    uint32_t koff[kDma], voff[kDma];
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
        const int r = drow_of(i);
        koff[i] = (uint32_t)(r * a.kv.token_stride) + 16u * (uint32_t)(dpos ^ k_swz<E4M3>(r));
        voff[i] = (uint32_t)(r * a.kv.token_stride) + 16u * (uint32_t)(dpos ^ v_swz<E4M3>(r));
    }
    const int32_t* row = a.kv.page_table + s.b * a.kv.table_stride;
    const int page_mask = (1 << a.kv.page_shift) - 1;
    // stage n of this wave: kTiles tiles from position stage_pos(n)
    auto stage_pos = [&](int n) { return p0 + (n * kWaves + wave) * F::kTiles * kPagedTile; };
    const int nstage = max(0, (p1 - p0 - wave * F::kTiles * kPagedTile + F::kUnit * kPagedTile - 1) /
                                  (F::kUnit * kPagedTile));
    // position of tile t of stage n; a stage's second tile may lie past the end: it then reads the first
    // one's rows again, masked
    auto tile_pos = [&](int n, int t) {
        const int pos = stage_pos(n);
        return pos + t * kPagedTile < p1 ? pos + t * kPagedTile : pos;
    };
    struct Ids {
        int id[F::kTiles];
    };
    auto page_ids = [&](int n) {
        Ids ids;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) ids.id[t] = load_const(row + (tile_pos(n, t) >> a.kv.page_shift));
        return ids;
    };
    auto issue = [&](int n, const Ids& ids) {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            const int pos = tile_pos(n, t);
            const int page = checked_page(ids.id[t], a.kv.n_pages, &bad);
            const int64_t off = page * a.kv.page_stride + kvh * a.kv.head_stride +
                                (int64_t)(pos & page_mask) * a.kv.token_stride;
            const uint8_t *kb = a.kv.k_pages + off, *vb = a.kv.v_pages + off;
            const uint32_t ls = lds0 + (uint32_t)((wave * kStages + (n & 1)) * kStage + t * F::kTile);
            if (pos + kPagedTile <= p1) {
#pragma unroll
                for (int i = 0; i < kDma; ++i) dma16_lds(kb, koff[i], ls + i * 1024);
#pragma unroll
                for (int i = 0; i < kDma; ++i) dma16_lds(vb, voff[i], ls + F::kTiles * F::kTile + i * 1024);
            } else {
                // rows past the last position read that position's: what lies there may be NaN, and
                // 0 * NaN would reach the sums
#pragma unroll
                for (int i = 0; i < kDma; ++i) {
                    const int r = drow_of(i), v = min(r, p1 - 1 - pos) * (int)a.kv.token_stride;
                    dma16_lds(kb, (uint32_t)v + 16u * (uint32_t)(dpos ^ k_swz<E4M3>(r)), ls + i * 1024);
                    dma16_lds(vb, (uint32_t)v + 16u * (uint32_t)(dpos ^ v_swz<E4M3>(r)),
                              ls + F::kTiles * F::kTile + i * 1024);
                }
            }
        }
    };
    // LDS reads: K's row l16; V^T's source row of this lane and its 8 bytes (see the head of the file)
    const int vrow = 4 * g + (l16 >> 2);
    auto read_v = [&](const uint8_t* tile, int b) {
        const int c = (2 * b + ((l16 & 3) >> 1)) ^ v_swz<E4M3>(vrow);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(tile + vrow * F::kRow + 16 * c + 8 * (l16 & 1)));
    };

    const float sc = a.scale2 * (E4M3 && a.kv.k_scale ? load_const(a.kv.k_scale + kvh) : 1.f);
    const float lazy = kLazy / sc;
    float m = -FLT_MAX, l = 0.f;                    // of head l16 (l: this lane's positions)
    f32x4 oacc[8];                                  // O^T: 8 blocks of 16 dims x 16 heads
#pragma unroll
    for (int b = 0; b < 8; ++b) oacc[b] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int n) {
        const uint8_t* kt = lds + (wave * kStages + (n & 1)) * kStage;
        const uint8_t* vt = kt + F::kTiles * F::kTile;
        f32x4 st[F::kTiles];
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint8_t* kr = kt + t * F::kTile + l16 * F::kRow;
            if constexpr (E4M3) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 c = load16(kr + 16 * ((4 * i + g) ^ k_swz<true>(l16)));
                    const uint2 c0 = e4m3x4_to_bf16(c.x), c1 = e4m3x4_to_bf16(c.y);
                    const uint2 c2 = e4m3x4_to_bf16(c.z), c3 = e4m3x4_to_bf16(c.w);
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{c0.x, c0.y, c1.x, c1.y}), qf[2 * i], st[t], 0, 0, 0);
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{c2.x, c2.y, c3.x, c3.y}), qf[2 * i + 1], st[t], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, load16(kr + 16 * ((4 * i + g) ^ k_swz<false>(l16)))), qf[i], st[t], 0,
                        0, 0);
            }
        }
        // Positions past the end.  No branch here: this compiler leaves out the wait between a matrix
        // product and a vector read of its result where a branch lies between them (a test looks for it).
        const int left = p1 - stage_pos(n) - 4 * g;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[t][i] = kPagedTile * t + i < left ? st[t][i] : -INFINITY;
        float top = fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3]));
        if constexpr (F::kTiles == 2)
            top = fmaxf(top, fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
        if (__builtin_amdgcn_ballot_w64(top > m + lazy)) {
            top = fmaxf(top, __shfl_xor(top, 16));              // the head's four lanes keep one maximum
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = top > m + lazy ? top : m;
            const float corr = fexp2((m - mn) * sc);
            l *= corr;
#pragma unroll
            for (int b = 0; b < 8; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) oacc[b][i] *= corr;
            m = mn;
        }
        const float mc = m * sc;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = fexp2(__builtin_fmaf(st[t][i], sc, -mc));
            l += (p[0] + p[1]) + (p[2] + p[3]);
            const uint32_t h01 = pack_bf16(p[0], p[1]), h23 = pack_bf16(p[2], p[3]);
            const uint32_t l01 = pack_bf16(p[0] - bf16lo_to_f32(h01), p[1] - bf16hi_to_f32(h01));
            const uint32_t l23 = pack_bf16(p[2] - bf16lo_to_f32(h23), p[3] - bf16hi_to_f32(h23));
            const bf16x8 w = __builtin_bit_cast(bf16x8, uint4{h01, h23, l01, l23});
            const uint8_t* tile = vt + t * F::kTile;
            if constexpr (E4M3) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    // positions 4 g .. + 3 of dims 32 b + 2 l16, + 1 as pairs of codes
                    const uint2 c = __builtin_bit_cast(uint2, read_v(tile, b));
                    const uint2 e = e4m3x4_to_bf16(__builtin_amdgcn_perm(c.y, c.x, 0x06040200u));
                    const uint2 o = e4m3x4_to_bf16(__builtin_amdgcn_perm(c.y, c.x, 0x07050301u));
                    oacc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{e.x, e.y, e.x, e.y}), w, oacc[2 * b], 0, 0, 0);
                    oacc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{o.x, o.y, o.x, o.y}), w, oacc[2 * b + 1], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    const uint2 v = __builtin_bit_cast(uint2, read_v(tile, b));
                    oacc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{v.x, v.y, v.x, v.y}), w, oacc[b], 0, 0, 0);
                }
            }
        }
    };

    Ids ids{}, next{};
    if (nstage > 0) ids = page_ids(0);
    if (nstage > 1) next = page_ids(1);
    // the query's loads done, so that the counts below are the DMAs' alone
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(qf[i]));
    if (nstage > 0) issue(0, ids);
    if (nstage > 1) issue(1, next);
    for (int n = 0; n < nstage; ++n) {
        const bool more = n + 2 < nstage;
        if (more) ids = page_ids(n + 2);                        // arrives under the wait and the products
        // stage n landed: at most stage n + 1's eight DMAs are still on their way
        if (n + 1 < nstage) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) asm volatile("" : "+s"(ids.id[t]));     // (not loaded later)
        compute(n);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its LDS reads returned before the refill
            issue(n + 2, ids);
        }
    }

    // the waves' results meet in LDS, in place of the stages
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float* sm_o = reinterpret_cast<float*>(lds);                    // [kWaves][kCols][kD]
    float* sm_m = sm_o + kWaves * kCols * kD;                       // [kWaves][kCols]
    float* sm_l = sm_m + kWaves * kCols;
    static_assert((kWaves * kCols * (kD + 2)) * 4 <= kLds, "merge space");
    __syncthreads();
    if (l16 < nrow) {
        if (g == 0) {
            sm_m[wave * kCols + l16] = m;
            sm_l[wave * kCols + l16] = bad ? NAN : l;
        }
        float* o = sm_o + (wave * kCols + l16) * kD;
#pragma unroll
        for (int b = 0; b < 8; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[E4M3 ? 32 * (b >> 1) + 2 * (4 * g + i) + (b & 1) : 16 * b + 4 * g + i] = oacc[b][i];
    }
    __syncthreads();
    if (bad && lane == 0 && a.kv.error)
        __hip_atomic_store(a.kv.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    const float vs = E4M3 && a.kv.v_scale ? load_const(a.kv.v_scale + kvh) : 1.f;
    for (int it = tid; it < nrow * (kD / 2); it += 64 * kWaves) {
        const int r = it / (kD / 2), d = it % (kD / 2) * 2;
        float M = sm_m[r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm_m[w * kCols + r]);
        float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float c = fexp2((sm_m[w * kCols + r] - M) * sc);
            const float2 o = *reinterpret_cast<const float2*>(sm_o + (w * kCols + r) * kD + d);
            L = __builtin_fmaf(sm_l[w * kCols + r], c, L);
            o0 = __builtin_fmaf(o.x, c, o0);
            o1 = __builtin_fmaf(o.y, c, o1);
        }
        const int h = head0 + r;
        if (s.nsplit == 1) {
            const float inv = L == 0.f ? 0.f : vs / L;
            *reinterpret_cast<uint32_t*>(a.o + (int64_t)s.b * a.ldo + (int64_t)h * kD + d) =
                pack_bf16(o0 * inv, o1 * inv);
        } else {
            const int64_t i = (int64_t)blockIdx.x * a.H + h;
            *reinterpret_cast<float2*>(a.part_o + i * kD + d) = float2{o0, o1};
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * i) = float2{M * sc, L};
        }
    }
}

// The splits of one (sequence, head) joined: O = sum_i c_i o_i / sum_i c_i l_i, c_i = 2^(m_i - max m).
// Wave w takes splits w, w + 4, ..; lane j dims 2 j, 2 j + 1.
__global__ __launch_bounds__(64 * kWaves) void sdpa_decode_paged_join_kernel(const PagedDecodeArgs a, int unit) {
    __shared__ float sm_m[kWaves], sm_l[kWaves];
    __shared__ float2 sm_o[kWaves][kD / 2];
    const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int nsplit;
    const int first = first_slot(a, b, plan_chunk(a, unit, lane), lane, &nsplit);
    if (nsplit == 1) return;
    float M = -FLT_MAX, L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 4
    for (int i = wave; i < nsplit; i += kWaves) {
        const int64_t p = (int64_t)(first + i) * a.H + h;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
        const float2 o = *reinterpret_cast<const float2*>(a.part_o + p * kD + 2 * lane);
        const float mn = fmaxf(M, ml.x);
        const float c = fexp2(M - mn), w = fexp2(ml.x - mn);
        L = __builtin_fmaf(w, ml.y, L * c);
        o0 = __builtin_fmaf(w, o.x, o0 * c);
        o1 = __builtin_fmaf(w, o.y, o1 * c);
        M = mn;
    }
    if (lane == 0) sm_m[wave] = M, sm_l[wave] = L;
    sm_o[wave][lane] = float2{o0, o1};
    __syncthreads();
    if (tid < kD / 2) {
        const float Mt = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
        L = o0 = o1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float c = fexp2(sm_m[w] - Mt);
            L = __builtin_fmaf(sm_l[w], c, L);
            o0 = __builtin_fmaf(sm_o[w][tid].x, c, o0);
            o1 = __builtin_fmaf(sm_o[w][tid].y, c, o1);
        }
        const float inv = (a.kv.v_scale ? a.kv.v_scale[h / a.group] : 1.f) / L;
        *reinterpret_cast<uint32_t*>(a.o + (int64_t)b * a.ldo + (int64_t)h * kD + 2 * tid) = pack_bf16(o0 * inv, o1 * inv);
    }
}

template <bool E4M3>
hipError_t launch(const PagedDecodeArgs& a, hipStream_t stream) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&sdpa_decode_paged_kernel<E4M3>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return attr;
    const dim3 grid(a.batch + a.budget, a.kv.n_kv, (a.group + kCols - 1) / kCols);
    hipLaunchKernelGGL(sdpa_decode_paged_kernel<E4M3>, grid, dim3(64 * kWaves), kLds, stream, a);
    const hipError_t e = hipGetLastError();
    // no sequence can have a second split where one split holds all that a row of the page table does
    if (e != hipSuccess || ((int64_t)a.kv.max_pages << a.kv.page_shift) <= Form<E4M3>::kUnit * kPagedTile) return e;
    hipLaunchKernelGGL(sdpa_decode_paged_join_kernel, dim3(a.batch, a.H), dim3(64 * kWaves), 0, stream, a,
                       Form<E4M3>::kUnit);
    return hipGetLastError();
}

}  // namespace

int sdpa_decode_paged_budget(int batch, int n_kv, int group) {
    (void)batch;
    const int per = n_kv * ((group + kCols - 1) / kCols);       // workgroups per split of a sequence
    return std::max(1, 2 * device_info().num_cu / per);         // two are resident on a CU
}

size_t sdpa_decode_paged_workspace_bytes(int batch, int n_heads, int n_kv) {
    const size_t slots = (size_t)batch + sdpa_decode_paged_budget(batch, n_kv, n_heads / n_kv);
    return slots * n_heads * (kD + 2) * sizeof(float);
}

hipError_t launch_sdpa_decode_paged(PagedDecodeArgs a, bool e4m3, void* workspace, hipStream_t stream) {
    a.budget = sdpa_decode_paged_budget(a.batch, a.kv.n_kv, a.group);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)(a.batch + a.budget) * a.H * kD;
    return e4m3 ? launch<true>(a, stream) : launch<false>(a, stream);
}

}  // namespace nmi
