// nmi_packed.hpp -- device side: which sequence and which piece of its new positions a workgroup works on, found
// from packed offsets in device memory.
#pragma once

#include "nmi_device.hpp"
#include "nmi_launch.hpp"

namespace nmi {

__device__ __forceinline__ void report(uint32_t* error) {
    if (error) __hip_atomic_store(error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Reports packed offsets out of order or range.  A wave's.
__device__ __forceinline__ void check_offsets(const int32_t* cu, int batch, int tokens, uint32_t* error, int lane) {
    bool bad = false;
    for (int i = lane; i < batch; i += 64) {
        int first;
        checked_span(cu[i], cu[i + 1], tokens, &first, &bad);
    }
    if (bad) report(error);
}

// New positions of sequence b: `rows` of them from `pos` on, row `row` of the packed ones the first; the piece asked
// for is the k-th of the sequence.
struct Packed {
    int b, row, rows;
    int64_t pos;
    uint32_t k;
};
// Piece x of all, where pieces(pos, rows) is a sequence's count; false where there are fewer.  64 sequences at a time
// in the lanes of the wave, all of which have to be active.
template <class PIECES>
__device__ __forceinline__ bool find_packed(const int32_t* cu, const int32_t* start_pos, int batch, int tokens, uint32_t x, int lane,
                                            PIECES pieces, Packed* found) {
    uint32_t upto = 0, end = 0;         // of the sequences before those in the lanes: pieces, and the end of their rows
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const int i = min(b0 + lane, batch - 1);
        const int c0 = cu[i], c1 = cu[i + 1], start = start_pos[i];
        bool bad = false;
        int first, place, rows = checked_span(c0, c1, tokens, &first, &bad);
        const uint32_t ends = max(wave_scan_max_u32(rows > 0 ? (uint32_t)(first + rows) : 0u), end);
        const uint32_t shifted = (uint32_t)__shfl_up((int)ends, 1);
        rows = later_span(c0, c1, tokens, (int)(lane ? shifted : end), &first, &place, &bad);
        const uint32_t mine = start < 0 || b0 + lane >= batch ? 0u : (uint32_t)pieces((int64_t)start + place, rows);
        const uint32_t at = upto + wave_scan_u32(mine);
        if (const uint64_t past = __builtin_amdgcn_ballot_w64(at > x)) {
            const int who = __builtin_ctzll(past);
            found->b = b0 + who;
            found->row = (int)lane_u32((uint32_t)first, who);
            found->rows = (int)lane_u32((uint32_t)rows, who);
            found->pos = (int64_t)(int)lane_u32((uint32_t)start, who) + (int)lane_u32((uint32_t)place, who);
            found->k = x - (lane_u32(at, who) - lane_u32(mine, who));
            return true;
        }
        upto = lane_u32(at, 63);
        end = lane_u32(ends, 63);
    }
    return false;
}

}  // namespace nmi
