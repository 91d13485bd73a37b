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
// Split: the tiles of 16 positions of all sequences, in a row, are dealt in equal shares to as many
// waves per KV head as are resident at once (range_tiles).  The lengths are read on the device: a scan
// over them tells a wave where its share begins, in which sequence.  So the launch depends on the
// batch size only, a captured graph stays right and balanced as the sequences grow, and a wave's load
// does not depend on how the positions are spread over the sequences.  The four waves of a workgroup
// whose tiles are all one sequence's take them in turn and add up their parts at the end: one piece
// (pieces_of).  A piece that is the whole of its sequence is finished where it is made; the others leave
// (maximum, row sum, sums), which a second kernel joins in a fixed order.
//
// Wave: stages of 8 KiB (16 positions of bf16, 32 of e4m3) brought into the wave's own LDS by DMA, one
// on its way while another is used, on past the end of a piece into the next sequence; waves wait for
// one another only to add up their parts.  A tile of 16 positions lies within a page: its address is one
// scalar.  Per tile:
// * S^T = K . Q^T (positions x heads) by 16x16x32 products: a lane then holds 4 positions of one head.
// * weights in base 2 against a running maximum that is raised only when a score exceeds it by 2^8
//   in weight, so that the sums are rarely rescaled.
// * O^T += V^T . P^T.  V^T comes from the token-major tile by transposing LDS reads.  bf16: the 32 places
//   of the product's inner dimension are the tile's 16 positions twice, with the weights' hi and lo
//   parts.  e4m3: the 16 positions of both tiles of a stage, one product for hi, one for lo; the
//   reads transpose pairs of dims, whose bytes are then sorted: the even dims of a block go to one
//   product, the odd ones to the next.
//
// Measured (graph replays, both launches; 40 query, 8 KV heads): one sequence of 777 positions 8.4 us, of
// 65536 45 (6.0 TB/s of the cache's bytes; a streaming read of as many 6.5); e4m3, 131072 positions 48.5
// (5.5); 64 of 90 to 8000 positions, e4m3, 48.6 (4.9); 128 of 500 48.4 (5.4).  What is left of a long one is the
// second launch and the gap before it (5 us), of a short one the two launches and the lengths, the
// page's id and the tile read one after another.
// Both sides of the choices, at 268 MB of cache: DMA past the caches 44 us, through them 50; eight waves per
// CU 44, ten with smaller stages 47; a workgroup's waves at separate shares throughout 44, and in turns over one
// 44 where the sequences are long but 56 where they are many (hence both, by is_joint).
#include "nmi_device.hpp"
#include "nmi_launch.hpp"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace nmi {

namespace {

constexpr int kD = kPagedHead;
constexpr int kWaves = kPagedWaves;
constexpr int kWgs = 2;                         // workgroups per CU
constexpr int kStage = 8192;                    // bytes of K and V per stage
constexpr int kStages = 2;                      // per wave
constexpr int kCols = 16;                       // query heads per wave
constexpr int kLds = kWaves * kStages * kStage;  // the stages; afterwards the waves' parts
static_assert(kWgs * kLds <= 160 * 1024 && kWaves * kCols * (kD + 2) * 4 <= kLds, "LDS");
constexpr float kLazy = 8.f;                    // log2 of the largest unnormalised weight

__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The row of all sequences' tiles, 64 sequences at a time in the lanes: those from b0 on, and the tiles
// of theirs and of all before them, up to each.
struct Lanes {
    int b0, len;
    uint32_t tiles, upto;
    bool bad;
};
__device__ __forceinline__ Lanes load_lanes(const PagedDecodeArgs& a, int b0, uint32_t before, int lane) {
    Lanes v;
    v.b0 = b0;
    v.bad = false;
    v.len = b0 + lane < a.batch ? checked_len(a.lens[b0 + lane], a.kv.max_pages, a.kv.page_shift, &v.bad) : 0;
    v.tiles = (uint32_t)(v.len + kPagedTile - 1) / kPagedTile;
    v.upto = before + wave_scan_u32(v.tiles);
    return v;
}

__device__ __forceinline__ uint32_t tiles_at(const PagedDecodeArgs& a, int b) {
    bool bad = false;
    const int len = a.lens[min(b, a.batch - 1)];
    return b < a.batch ? (uint32_t)(checked_len(len, a.kv.max_pages, a.kv.page_shift, &bad) + kPagedTile - 1) / kPagedTile : 0u;
}

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

template <bool E4M3>
struct Form {
    static constexpr int kTiles = E4M3 ? 2 : 1;         // per stage
    static constexpr int kRow = E4M3 ? kD : 2 * kD;     // bytes of a position
    static constexpr int kTile = kPagedTile * kRow;
};

// LDS tiles: row r of 16-byte chunks, chunk c at c ^ swz(r), so that the reads of 16 rows at one chunk
// (K) or at one 32-byte column (V) spread over the banks.
template <bool E4M3>
__device__ __forceinline__ int k_swz(int r) { return E4M3 ? (r >> 1) & 7 : r & 15; }
template <bool E4M3>
__device__ __forceinline__ int v_swz(int r) { return E4M3 ? 2 * ((r >> 1) & 3) : 2 * (r & 7); }

// A stage on its way: positions [pos, pos + 16 kTiles), cut at `stop`, of sequence b; whether it begins
// and ends its piece, and whether the piece is the whole sequence.
struct Stage {
    int b, pos, stop;
    bool valid, first, last, whole;
    bool overlong, bad;     // the length is more than the table holds; a page that the pool does not have
    bf16x8 q[4];            // of a first one: this lane's head as the B operand
};

// MANY: more sequences than lanes.
template <bool E4M3, bool MANY>
__global__ __launch_bounds__(64 * kWaves, 2) void sdpa_decode_paged_kernel(const PagedDecodeArgs a) {
    typedef Form<E4M3> F;
    typedef __attribute__((address_space(3))) void lds_void;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y, r0 = blockIdx.z * kCols, nrow = min(kCols, a.group - r0);
    const int head0 = kvh * a.group + r0;
    const uint32_t me = blockIdx.x * kWaves + wave;

    // this wave's tiles, and the sequence that they begin in
    Lanes v = load_lanes(a, 0, 0, lane);
    uint32_t total = lane_u32(v.upto, 63);
    if constexpr (MANY) {
        uint32_t tiles = v.tiles;
        for (int b0 = 64; b0 < a.batch; b0 += 4 * 64)           // (lengths of four times 64 on their way at once)
#pragma unroll
            for (int c = 0; c < 4; ++c) tiles += tiles_at(a, b0 + 64 * c + lane);
        total = lane_u32(wave_scan_u32(tiles), 63);
    }
    const int c = range_tiles(total, a.waves, F::kTiles);
    if (me + 1 == (uint32_t)a.waves && kvh == 0 && r0 == 0) {
        // for the joining kernel (the last wave: the first to have no tiles)
        for (Lanes w = v;; w = load_lanes(a, w.b0 + 64, lane_u32(w.upto, 63), lane)) {
            const Pieces p = w.tiles ? pieces_of(w.upto - w.tiles, w.tiles, c, total) : Pieces{};
            if (w.b0 + lane < a.batch) a.plan[w.b0 + lane] = p;
            if (!MANY || w.b0 + 64 >= a.batch) break;
        }
    }
    // the first sequence with tiles past `at`: its lane; 64 where there is none (only if the lengths change
    // under the launch)
    auto seek = [&](uint32_t at) {
        if constexpr (MANY)
            while (look_on(at, lane_u32(v.upto, 63), v.b0, a.batch))
                v = load_lanes(a, v.b0 + 64, lane_u32(v.upto, 63), lane);
        return __popcll(__builtin_amdgcn_ballot_w64(v.upto <= at));
    };
    uint32_t at = range_first(blockIdx.x * kWaves, c, total), end = range_first((blockIdx.x + 1) * kWaves, c, total);
    if (at >= end) return;
    int i = seek(at);
    if (MANY && i == 64) return;
    const bool joint = is_joint(blockIdx.x, lane_u32(v.upto - v.tiles, i), lane_u32(v.tiles, i), c, total);
    if (!joint) {
        at = range_first(me, c, total);
        end = range_first(me + 1, c, total);
        if (at >= end) return;
        i = seek(at);
        if (MANY && i == 64) return;
    }
    constexpr int kStep = F::kTiles * kPagedTile;               // positions of a stage
    const int stride = joint ? kWaves * kStep : kStep;          // from one of a wave's stages to its next

    const float sc = a.scale2 * (E4M3 && a.kv.k_scale ? load_const(a.kv.k_scale + kvh) : 1.f);
    const float vs = E4M3 && a.kv.v_scale ? load_const(a.kv.v_scale + kvh) : 1.f;
    const float lazy = kLazy / sc;
    // the maximum of nothing: times sc still finite
    const float lowest = sc > 1.f ? -0x1p127f * __builtin_amdgcn_rcpf(sc) : -FLT_MAX;
    const int page_mask = (1 << a.kv.page_shift) - 1;
    const int64_t head_off = kvh * a.kv.head_stride;

    // DMA: instruction k brings 1 KiB, rows r = (1024 / kRow) k + lane / (kRow / 16) of a tile
    constexpr int kChunks = F::kRow / 16, kDma = F::kTile / 1024;        // per row; per tile
    const int drow = lane / kChunks, dpos = lane % kChunks;
    auto drow_of = [&](int k) { return drow + (64 / kChunks) * k; };
    uint32_t koff[kDma], voff[kDma];
#pragma unroll
    for (int k = 0; k < kDma; ++k) {
        const int r = drow_of(k);
        koff[k] = (uint32_t)(r * a.kv.token_stride) + 16u * (uint32_t)(dpos ^ k_swz<E4M3>(r));
        voff[k] = (uint32_t)(r * a.kv.token_stride) + 16u * (uint32_t)(dpos ^ v_swz<E4M3>(r));
    }

    // --- the producer: the next stage's place, its page ids already asked for
    struct {
        int b, pos, stop;
        bool first, whole, bad;
        const int32_t* row;
        int id[F::kTiles];
    } nx;
    auto ask = [&]() {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            // (a stage's second tile may lie past the end: it reads the first one's rows again, masked)
            const int p = nx.pos + t * kPagedTile < nx.stop ? nx.pos + t * kPagedTile : nx.pos;
            nx.id[t] = load_const(nx.row + (p >> a.kv.page_shift));
        }
    };
    auto open_piece = [&]() {       // the piece that begins at tile `at`, in lane i's sequence
        const uint32_t tiles = lane_u32(v.tiles, i), first = lane_u32(v.upto, i) - tiles;
        const uint32_t stop = min(end, first + tiles);
        nx.b = v.b0 + i;
        nx.pos = (int)(at - first) * kPagedTile + (joint ? wave * kStep : 0);
        nx.stop = min((int)lane_u32((uint32_t)v.len, i), (int)(stop - first) * kPagedTile);
        nx.first = true;
        nx.whole = stop - at == tiles;
        nx.bad = (__builtin_amdgcn_ballot_w64(v.bad) >> i) & 1;
        nx.row = a.kv.page_table + nx.b * a.kv.table_stride;
        at = stop;
        if (nx.pos < nx.stop) ask();
    };
    auto advance = [&]() {          // past the stage just issued; false at the end of this wave's tiles
        nx.first = false;
        nx.pos += stride;
        if (nx.pos < nx.stop) {
            ask();
            return true;
        }
        if (at >= end) return false;
        i = seek(at);
        if (MANY && i == 64) return false;
        open_piece();
        return true;
    };
    open_piece();
    const int piece_b = nx.b, piece_pos = nx.pos, piece_stop = nx.stop;    // (of a joint one)
    const bool piece_whole = nx.whole;
    bool bad = nx.bad;
    bool more = nx.pos < nx.stop;       // (a joint piece may have no stage for this wave)
    auto issue = [&](int slot, Stage& s) __attribute__((always_inline)) {
        s.valid = more;
        if (!more) return;
        s.b = nx.b, s.pos = nx.pos, s.stop = nx.stop;
        s.first = nx.first, s.whole = nx.whole, s.overlong = nx.bad, s.bad = false;
        if (nx.first) {
            // of a bf16 cache, step k holds dims 32 k + 8 g .. + 7; of an e4m3 cache, steps 2 k and 2 k + 1
            // dims 64 k + 16 g .. + 15 (one 16-byte read of K)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = E4M3 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
                const int h = head0 + min(l16, nrow - 1);               // (unused columns: any head)
                s.q[k] = __builtin_bit_cast(bf16x8, load16(a.q + (int64_t)nx.b * a.ldq + (int64_t)h * kD + d));
            }
        }
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            const int pos = nx.pos + t * kPagedTile < nx.stop ? nx.pos + t * kPagedTile : nx.pos;
            const int page = checked_page(nx.id[t], a.kv.n_pages, &s.bad);
            const int64_t off = page * a.kv.page_stride + head_off + (int64_t)(pos & page_mask) * a.kv.token_stride;
            const uint8_t *kb = a.kv.k_pages + off, *vb = a.kv.v_pages + off;
            const uint32_t ls = lds0 + (uint32_t)((wave * kStages + slot) * kStage + t * F::kTile);
            constexpr int kV = F::kTiles * F::kTile;
            if (pos + kPagedTile <= nx.stop) {
#pragma unroll
                for (int k = 0; k < kDma; ++k) dma16_lds_nt(kb, koff[k], ls + k * 1024);
#pragma unroll
                for (int k = 0; k < kDma; ++k) dma16_lds_nt(vb, voff[k], ls + kV + k * 1024);
            } else {
                // rows past the last position read that position's: what lies there may be NaN, and
                // 0 * NaN would reach the sums
#pragma unroll
                for (int k = 0; k < kDma; ++k) {
                    const int r = drow_of(k), u = min(r, nx.stop - 1 - pos) * (int)a.kv.token_stride;
                    dma16_lds_nt(kb, (uint32_t)u + 16u * (uint32_t)(dpos ^ k_swz<E4M3>(r)), ls + k * 1024);
                    dma16_lds_nt(vb, (uint32_t)u + 16u * (uint32_t)(dpos ^ v_swz<E4M3>(r)), ls + kV + k * 1024);
                }
            }
        }
        more = advance();
        s.last = !more || nx.first;
    };

    // --- the consumer
    // V^T's source row of this lane and its 8 bytes: output lane 4 a + b, element e of a transposing read
    // is element b of source lane 4 e + a's 8 bytes, in each 16 lanes
    const int vrow = 4 * g + (l16 >> 2);
    auto read_v = [&](const uint8_t* tile, int b) {
        const int ch = (2 * b + ((l16 & 3) >> 1)) ^ v_swz<E4M3>(vrow);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(tile + vrow * F::kRow + 16 * ch + 8 * (l16 & 1)));
    };
    bf16x8 qf[4];
    int from = 0;                                   // the piece's first position
    float m = lowest, l = 0.f;                      // of head l16 (l: this lane's positions)
    f32x4 oacc[8];                                  // O^T: 8 blocks of 16 dims x 16 heads
#pragma unroll
    for (int b = 0; b < 8; ++b) oacc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int slot, const Stage& s) __attribute__((always_inline)) {
        const uint8_t* kt = lds + (wave * kStages + slot) * kStage;
        const uint8_t* vt = kt + F::kTiles * F::kTile;
        constexpr int kFrags = E4M3 ? 4 : 8;                    // of V^T, per tile
        f32x4 st[F::kTiles];
        uint2 vf[F::kTiles][kFrags];
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint8_t* kr = kt + t * F::kTile + l16 * F::kRow;
            if constexpr (E4M3) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 w = load16(kr + 16 * ((4 * k + g) ^ k_swz<true>(l16)));
                    const uint2 w0 = e4m3x4_to_bf16(w.x), w1 = e4m3x4_to_bf16(w.y);
                    const uint2 w2 = e4m3x4_to_bf16(w.z), w3 = e4m3x4_to_bf16(w.w);
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{w0.x, w0.y, w1.x, w1.y}), qf[2 * k], st[t], 0, 0, 0);
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, uint4{w2.x, w2.y, w3.x, w3.y}), qf[2 * k + 1], st[t], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, load16(kr + 16 * ((4 * k + g) ^ k_swz<false>(l16)))), qf[k], st[t], 0,
                        0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t)
#pragma unroll
            for (int b = 0; b < kFrags; ++b) vf[t][b] = __builtin_bit_cast(uint2, read_v(vt + t * F::kTile, b));
        // Positions past the end.  No branch here: this compiler leaves out the wait between a matrix
        // product and a vector read of its result where a branch lies between them (a test looks for it).
        const int left = s.stop - s.pos - 4 * g;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) st[t][k] = kPagedTile * t + k < left ? st[t][k] : -INFINITY;
        float top = fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3]));
        if constexpr (F::kTiles == 2)
            top = fmaxf(top, fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
        if (__builtin_amdgcn_ballot_w64(top > m + lazy)) {
            top = rows_max(top);                                // the head's four lanes keep one maximum
            const float mn = top > m + lazy ? top : m;
            const float corr = fexp2((m - mn) * sc);
            l *= corr;
#pragma unroll
            for (int b = 0; b < 8; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) oacc[b][k] *= corr;
            m = mn;
        }
        const float mc = m * sc;
        uint32_t hi[F::kTiles][2], lo[F::kTiles][2];            // the weights of each tile's 4 positions
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            float p[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = fexp2(__builtin_fmaf(st[t][k], sc, -mc));
            l += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                hi[t][k] = pack_bf16(p[2 * k], p[2 * k + 1]);
                lo[t][k] = pack_bf16(p[2 * k] - bf16lo_to_f32(hi[t][k]), p[2 * k + 1] - bf16hi_to_f32(hi[t][k]));
            }
        }
        auto frag = [](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
            return __builtin_bit_cast(bf16x8, uint4{a0, a1, a2, a3});
        };
        if constexpr (E4M3) {
            const bf16x8 wh = frag(hi[0][0], hi[0][1], hi[1][0], hi[1][1]);
            const bf16x8 wl = frag(lo[0][0], lo[0][1], lo[1][0], lo[1][1]);
#pragma unroll
            for (int b = 0; b < kFrags; ++b) {
                // positions 4 g .. + 3 of dims 32 b + 2 l16, + 1 of both tiles, as pairs of codes
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    const uint32_t pick = odd ? 0x07050301u : 0x06040200u;
                    const uint2 x0 = e4m3x4_to_bf16(__builtin_amdgcn_perm(vf[0][b].y, vf[0][b].x, pick));
                    const uint2 x1 = e4m3x4_to_bf16(__builtin_amdgcn_perm(vf[1][b].y, vf[1][b].x, pick));
                    const bf16x8 x = frag(x0.x, x0.y, x1.x, x1.y);
                    f32x4& acc = oacc[2 * b + odd];
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, wh, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, wl, acc, 0, 0, 0);
                }
            }
        } else {
            const bf16x8 w = frag(hi[0][0], hi[0][1], lo[0][0], lo[0][1]);
#pragma unroll
            for (int b = 0; b < kFrags; ++b)
                oacc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    frag(vf[0][b].x, vf[0][b].y, vf[0][b].x, vf[0][b].y), w, oacc[b], 0, 0, 0);
        }
    };
    // A piece's end.  A lane's sums are its head's dims 16 b + 4 g .. + 3 of block b (bf16), or 32 b + 8 g
    // .. + 7 alternating over blocks 2 b and 2 b + 1 (e4m3).
    auto dim = [&](int b) { return E4M3 ? 32 * (b >> 1) + 8 * g + 4 * (b & 1) : 16 * b + 4 * g; };
    auto four = [&](int b) {
        if constexpr (E4M3) {
            const int e = b & ~1, k = 2 * (b & 1);
            return f32x4{oacc[e][k], oacc[e + 1][k], oacc[e][k + 1], oacc[e + 1][k + 1]};
        } else {
            return oacc[b];
        }
    };
    auto row_sum = [&]() {
        if (bad && lane == 0 && a.kv.error)
            __hip_atomic_store(a.kv.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        const float L = rows_sum(l);
        return bad ? NAN : L;
    };
    // A value of v that is not finite makes NaN of its dim's sums by the weights' low parts (0 or negative), and
    // by the rows past the last position.  Its weight is positive, so that a dim's values that are not
    // finite, added up by themselves (an infinity, or NaN), are its sum: two dims a lane, over what the wave's
    // stages from `pos` to `stop` have of sequence b; 0 for other dims.  It takes the place of what was stored.
    // (The test of the sums costs 0.1 to 0.3 us of 8 to 50; an amended oacc in place of what was stored, which
    // the compiler keeps twice, cost 0.5.)
    auto odd_sums = [&]() __attribute__((always_inline)) -> bool {
        if constexpr (E4M3) return false;
        f32x4 sum = oacc[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) sum += oacc[i];
        const bool odd = !(fabsf((sum[0] + sum[1]) + (sum[2] + sum[3])) < INFINITY);
        return __builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0);
    };
    auto odd_values = [&](int b, int pos, int stop) __attribute__((always_inline)) {
        const int32_t* row = a.kv.page_table + b * a.kv.table_stride;
        float2 x{0.f, 0.f};
        for (; pos < stop; pos += stride) {
            bool none = false;          // (reported by the stage that met it)
            const int page = checked_page(load_const(row + (pos >> a.kv.page_shift)), a.kv.n_pages, &none);
            const uint8_t* vp = a.kv.v_pages + page * a.kv.page_stride + head_off + 4 * lane +
                                (int64_t)(pos & page_mask) * a.kv.token_stride;
#pragma unroll 4
            for (int r = min(kPagedTile, stop - pos); r > 0; --r, vp += a.kv.token_stride) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(vp);
                if ((w & 0x7F80u) == 0x7F80u) x.x += bf16lo_to_f32(w);
                if ((w & 0x7F800000u) == 0x7F800000u) x.y += bf16hi_to_f32(w);
            }
        }
        return x;
    };
    auto finish = [&](const Stage& s) __attribute__((always_inline)) {
        const float L = row_sum();
        const int h = head0 + l16;
        if (l16 >= nrow) {
        } else if (s.whole) {
            const float inv = vs / L;
            uint16_t* o = a.o + (int64_t)s.b * a.ldo + (int64_t)h * kD;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const f32x4 x = four(b);
                uint32_t* p = reinterpret_cast<uint32_t*>(o + dim(b));
                p[0] = pack_bf16(x[0] * inv, x[1] * inv);
                p[1] = pack_bf16(x[2] * inv, x[3] * inv);
            }
        } else {
            const int64_t slot = (int64_t)(me + s.b) * a.H + h;
#pragma unroll
            for (int b = 0; b < 8; ++b) *reinterpret_cast<f32x4*>(a.part_o + slot * kD + dim(b)) = four(b);
            if (g == 0) a.part_ml[slot] = float2{m * sc, L};
        }
        if (odd_sums()) {
            const float2 x = odd_values(s.b, from, s.stop);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // the stores above, by other lanes
#pragma unroll 1
            for (int r = 0; r < nrow; ++r) {
                const float Lr = __uint_as_float(lane_u32(__float_as_uint(L), r));
                if (s.whole) {
                    uint16_t* o = a.o + (int64_t)s.b * a.ldo + (int64_t)(head0 + r) * kD + 2 * lane;
                    if (x.x != 0.f && Lr == Lr) o[0] = (uint16_t)(__float_as_uint(x.x) >> 16);
                    if (x.y != 0.f && Lr == Lr) o[1] = (uint16_t)(__float_as_uint(x.y) >> 16);
                } else {
                    float* o = a.part_o + ((int64_t)(me + s.b) * a.H + head0 + r) * kD + 2 * lane;
                    if (x.x != 0.f) o[0] = x.x;
                    if (x.y != 0.f) o[1] = x.y;
                }
            }
        }
    };

    Stage stage[kStages];
#pragma unroll
    for (int k = 0; k < kStages; ++k) issue(k, stage[k]);
    for (;;) {
        // one stage of the ring: its DMAs landed (the other's eight, if it has any, may be on their way; stores
        // and loads of the code around only make the wait longer), used, refilled
        auto turn = [&](auto slot) __attribute__((always_inline)) {
            constexpr int k = decltype(slot)::value;
            Stage& s = stage[k];
            if (!s.valid) return false;
            if (stage[k ^ 1].valid) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (s.first) {
                m = lowest;
                l = 0.f;
                bad = s.overlong;
                from = s.pos;
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[j] = s.q[j];
#pragma unroll
                for (int b = 0; b < 8; ++b) oacc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            bad |= s.bad;
            compute(k, s);
            if (s.last && !joint) finish(s);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // its LDS reads returned before the refill
            issue(k, s);
            return true;
        };
        static_assert(kStages == 2, "the ring's two turns");
        if (!turn(std::integral_constant<int, 0>{})) break;
        if (!turn(std::integral_constant<int, 1>{})) break;
    }
    if (!joint) return;

    // a joint piece: the waves' parts (of one without a stage: nothing) meet in LDS, in place of the stages
    float* sm_o = reinterpret_cast<float*>(lds);                    // [kWaves][kCols][kD]
    float* sm_m = sm_o + kWaves * kCols * kD;                       // [kWaves][kCols]
    float* sm_l = sm_m + kWaves * kCols;
    const float L = row_sum();
    __syncthreads();
    if (l16 < nrow) {
#pragma unroll
        for (int b = 0; b < 8; ++b) *reinterpret_cast<f32x4*>(sm_o + (wave * kCols + l16) * kD + dim(b)) = four(b);
        if (g == 0) {
            sm_m[wave * kCols + l16] = m;
            sm_l[wave * kCols + l16] = L;
        }
    }
    if (odd_sums()) {
        const float2 x = odd_values(piece_b, piece_pos, piece_stop);
        __builtin_amdgcn_wave_barrier();        // (LDS writes of one wave are in order)
#pragma unroll 1
        for (int r = 0; r < nrow; ++r) {
            float* o = sm_o + (wave * kCols + r) * kD + 2 * lane;
            if (x.x != 0.f) o[0] = x.x;
            if (x.y != 0.f) o[1] = x.y;
        }
    }
    __syncthreads();
    for (int it = tid; it < nrow * (kD / 2); it += 64 * kWaves) {
        const int r = it / (kD / 2), d = it % (kD / 2) * 2, h = head0 + r;
        float M = sm_m[r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm_m[w * kCols + r]);
        float Ls = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = fexp2((sm_m[w * kCols + r] - M) * sc);
            const float2 o = *reinterpret_cast<const float2*>(sm_o + (w * kCols + r) * kD + d);
            Ls = __builtin_fmaf(sm_l[w * kCols + r], f, Ls);
            o0 = __builtin_fmaf(o.x, f, o0);
            o1 = __builtin_fmaf(o.y, f, o1);
        }
        if (piece_whole) {
            const float inv = vs / Ls;
            *reinterpret_cast<uint32_t*>(a.o + (int64_t)piece_b * a.ldo + (int64_t)h * kD + d) =
                pack_bf16(o0 * inv, o1 * inv);
        } else {
            const int64_t slot = (int64_t)(blockIdx.x * kWaves + piece_b) * a.H + h;
            *reinterpret_cast<float2*>(a.part_o + slot * kD + d) = float2{o0, o1};
            if (d == 0) a.part_ml[slot] = float2{M * sc, Ls};
        }
    }
}

// The pieces of a sequence's heads joined: O = sum_i c_i o_i / sum_i c_i l_i, c_i = 2^(m_i - max m); a
// sequence of one piece is done already, one of none gets zeros.  A workgroup takes `heads` heads.  Of
// few pieces, each wave joins a head by itself, two dims a lane; of many, all waves join one head after
// another: wave w dims 32 w .. + 31 of pieces lane / 8, + 8, .., four dims a lane, eight pieces of a lane on
// their way at once.  (With four at once and 16 waves to a head of few sequences: 777 positions 9.3 us
// both launches, 8.8 so; 60001 45.5, 46.2 so.)
constexpr int kFewPieces = 8, kAtOnce = 8;
__global__ __launch_bounds__(64 * kWaves) void sdpa_decode_paged_join_kernel(const PagedDecodeArgs a, int heads) {
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Pieces plan = a.plan[b];
    const int n = plan.count();
    if (n == 1) return;
    const int h0 = blockIdx.y * heads, h1 = min(h0 + heads, a.H);
    uint32_t* out = reinterpret_cast<uint32_t*>(a.o + (int64_t)b * a.ldo);
    auto slot = [&](int i, int h) { return (int64_t)(plan.owner(i) + b) * a.H + h; };
    if (n == 0) {
        for (int i = h0 * (kD / 2) + tid; i < h1 * (kD / 2); i += 64 * kWaves) out[i] = 0u;
        return;
    }
    if (n <= kFewPieces) {
        for (int h = h0 + wave; h < h1; h += kWaves) {
            const float2 ml = a.part_ml[slot(min(lane & (kFewPieces - 1), n - 1), h)];
            float2 o[kFewPieces];
#pragma unroll
            for (int i = 0; i < kFewPieces; ++i)
                if (i < n) o[i] = *reinterpret_cast<const float2*>(a.part_o + slot(i, h) * kD + 2 * lane);
            // (every 8 lanes hold the pieces, the last again where there are fewer)
            float M = fmaxf(ml.x, dpp_f32<0xB1>(ml.x));
            M = fmaxf(M, dpp_f32<0x4E>(M));
            M = fmaxf(M, dpp_f32<0x141>(M));
            const float c = fexp2(ml.x - M), cl = c * ml.y;     // of piece `lane`
            float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
            for (int i = 0; i < kFewPieces; ++i)
                if (i < n) {
                    const float ci = __uint_as_float(lane_u32(__float_as_uint(c), i));
                    L += __uint_as_float(lane_u32(__float_as_uint(cl), i));
                    o0 = __builtin_fmaf(ci, o[i].x, o0);
                    o1 = __builtin_fmaf(ci, o[i].y, o1);
                }
            const float inv = (a.kv.v_scale ? a.kv.v_scale[h / a.group] : 1.f) / L;
            out[h * (kD / 2) + lane] = pack_bf16(o0 * inv, o1 * inv);
        }
        return;
    }
    const int quad = 8 * wave + (lane & 7);
    for (int h = h0; h < h1; ++h) {
        float M = -FLT_MAX, L = 0.f;
        f32x4 o{0.f, 0.f, 0.f, 0.f};
        for (int i0 = lane >> 3; i0 < n; i0 += 8 * kAtOnce) {
            float2 ml[kAtOnce];
            f32x4 oi[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int i = i0 + 8 * k;
                ml[k] = float2{-FLT_MAX, 0.f};
                oi[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (i < n) {
                    const int64_t p = slot(i, h);
                    ml[k] = a.part_ml[p];
                    oi[k] = *reinterpret_cast<const f32x4*>(a.part_o + p * kD + 4 * quad);
                }
            }
            float mn = M;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
            const float c = fexp2(M - mn);
            L *= c;
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] *= c;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float w = fexp2(ml[k].x - mn);
                L = __builtin_fmaf(w, ml[k].y, L);
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] = __builtin_fmaf(w, oi[k][d], o[d]);
            }
            M = mn;
        }
        // over the lanes of the same dims (8 apart: the other half of the row, then the rows)
        const float mw = rows_max(fmaxf(M, dpp_f32<0x128>(M)));
        const float c = fexp2(M - mw);
        L = rows_sum(L * c + dpp_f32<0x128>(L * c));
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = rows_sum(o[d] * c + dpp_f32<0x128>(o[d] * c));
        if (lane < 8) {
            const float inv = (a.kv.v_scale ? a.kv.v_scale[h / a.group] : 1.f) / L;
            uint32_t* q = out + h * (kD / 2) + 2 * quad;
            q[0] = pack_bf16(o[0] * inv, o[1] * inv);
            q[1] = pack_bf16(o[2] * inv, o[3] * inv);
        }
    }
}

template <bool E4M3, bool MANY>
hipError_t launch(const PagedDecodeArgs& a, hipStream_t stream) {
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void*>(&sdpa_decode_paged_kernel<E4M3, MANY>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return attr;
    const dim3 grid(a.waves / kWaves, a.kv.n_kv, (a.group + kCols - 1) / kCols);
    hipLaunchKernelGGL((sdpa_decode_paged_kernel<E4M3, MANY>), grid, dim3(64 * kWaves), kLds, stream, a);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    // Many sequences are in few pieces each, most in one: workgroups that find nothing to do are what it costs.
    const int heads = std::min(8, (int)(((int64_t)a.batch * a.H + 2047) / 2048));
    hipLaunchKernelGGL(sdpa_decode_paged_join_kernel, dim3(a.batch, (a.H + heads - 1) / heads), dim3(64 * kWaves), 0, stream,
                       a, heads);
    return hipGetLastError();
}

struct Layout {
    size_t part_o, part_ml, plan, total;        // byte offsets
};
Layout layout(int batch, int n_heads, int waves) {
    const size_t slots = (size_t)batch + waves;
    Layout w{};
    w.part_ml = slots * n_heads * kD * sizeof(float);
    w.plan = w.part_ml + slots * n_heads * sizeof(float2);
    w.total = w.plan + (size_t)batch * sizeof(Pieces);
    return w;
}

}  // namespace

int sdpa_decode_paged_waves(int n_kv, int group) {
    const int per = n_kv * ((group + kCols - 1) / kCols);
    return std::max(1, kWgs * device_info().num_cu / per) * kWaves;
}

size_t sdpa_decode_paged_workspace_bytes(int batch, int n_heads, int n_kv) {
    return layout(batch, n_heads, sdpa_decode_paged_waves(n_kv, n_heads / n_kv)).total;
}

hipError_t launch_sdpa_decode_paged(PagedDecodeArgs a, bool e4m3, void* workspace, hipStream_t stream) {
    a.waves = sdpa_decode_paged_waves(a.kv.n_kv, a.group);
    const Layout w = layout(a.batch, a.H, a.waves);
    char* base = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(base + w.part_o);
    a.part_ml = reinterpret_cast<float2*>(base + w.part_ml);
    a.plan = reinterpret_cast<Pieces*>(base + w.plan);
    if (a.batch > 64) return e4m3 ? launch<true, true>(a, stream) : launch<false, true>(a, stream);
    return e4m3 ? launch<true, false>(a, stream) : launch<false, false>(a, stream);
}

}  // namespace nmi
