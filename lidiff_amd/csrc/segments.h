// Row ranges of a batch of scans ("segments": int32 [S][2], first row and the row behind the last one, ascending and disjoint; an
// empty range may name any row).
// Every kernel that works scan by scan cuts the rows into tiles that belong to ONE segment, so that no tile ever reads a row of
// another scan (whose values -- Inf, NaN -- could otherwise reach a product with a zero weight).
#pragma once
#include "common.h"

namespace lidiff {

struct SegTile {
    int seg;        // -1: rows that belong to no segment (in front of, between or behind the segments)
    int lo, hi;     // rows [lo, hi); lo == hi: nothing to do
};

// Workgroups a launch needs so that every row of [0, rows) has a tile: a segment and the gap in front of it each round up once.
inline int64_t seg_tiles_bound(int64_t rows, int per, const void* seg, int64_t nseg) {
    return ceil_div(rows, per) + (seg ? 2 * nseg + 1 : 0);
}

__device__ __forceinline__ int2 seg_range(const int32_t* __restrict__ seg, int s, int rows) {
    if (seg == nullptr) return make_int2(0, rows);
    const int2 r = reinterpret_cast<const int2*>(seg)[s];
    const int lo = min(max(r.x, 0), rows);              // whatever the ranges say, no row outside [0, rows) is touched
    return make_int2(lo, min(max(r.y, lo), rows));
}

// Tile number `tile` of the sequence gap 0, segment 0, gap 1, segment 1, ..., last gap, each cut every `per` rows.  One wave, all lanes
// active: a lane takes a segment, an inclusive scan of the tile counts over the wave finds the owner, 64 segments a round.
__device__ inline SegTile find_seg_tile(const int32_t* __restrict__ seg, int nseg, int rows, int per, int tile) {
    if (seg == nullptr) {
        const int64_t lo = (int64_t)tile * per;
        return lo < rows ? SegTile{0, (int)lo, (int)min((int64_t)rows, lo + per)} : SegTile{-1, 0, 0};
    }
    const int lane = lane_id();
    int before = 0, prev_end = 0;
    for (int base = 0; base <= nseg; base += kWave) {
        const int i = base + lane;
        const int2 r = i < nseg ? seg_range(seg, i, rows) : make_int2(rows, rows);
        const int own = (int)(((int64_t)r.y - r.x + per - 1) / per);
        int upto = own > 0 ? r.y : 0;                       // rows of the segments so far (an empty one may name any row)
        for (int off = 1; off < kWave; off <<= 1) {
            const int up = __shfl_up(upto, off);
            if (lane >= off) upto = max(upto, up);
        }
        upto = max(upto, prev_end);
        const int up1 = __shfl_up(upto, 1), pe = lane == 0 ? prev_end : up1;
        const int gap = (own > 0 || i == nseg) && r.x > pe ? (int)(((int64_t)r.x - pe + per - 1) / per) : 0;
        int incl = gap + own;
        for (int off = 1; off < kWave; off <<= 1) {
            const int up = __shfl_up(incl, off);
            if (lane >= off) incl += up;
        }
        const int excl = before + incl - gap - own;
        const unsigned long long hit = __ballot(tile >= excl && tile < excl + gap + own);
        if (hit) {
            const int src = __ffsll((long long)hit) - 1;
            const int t = tile - __shfl(excl, src), g = __shfl(gap, src), s0 = __shfl(r.x, src), e0 = __shfl(r.y, src),
                      p0 = __shfl(pe, src);
            SegTile out;
            if (t < g) out = SegTile{-1, p0 + t * per, min(s0, p0 + (t + 1) * per)};
            else out = SegTile{base + src, s0 + (t - g) * per, min(e0, s0 + (t - g + 1) * per)};
            out.seg = __builtin_amdgcn_readfirstlane(out.seg);
            out.lo = __builtin_amdgcn_readfirstlane(out.lo);
            out.hi = __builtin_amdgcn_readfirstlane(out.hi);
            return out;
        }
        before += __shfl(incl, kWave - 1);
        prev_end = __shfl(upto, kWave - 1);
    }
    return SegTile{-1, 0, 0};
}

}  // namespace lidiff
