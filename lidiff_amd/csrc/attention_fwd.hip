// Attention between the rows of the same scan, forward: out_i = sum_j softmax_j(q_i . k_j scale + bias_h(|c_i - c_j|)) v_j over the keys j of
// i's scan (segments.h), in one pass over the keys with a running base and sum per query and head.  A query whose scan has no keys, and a
// row of no scan, gives zeros.
//
// The base need not be the maximum: it follows a score that exceeds it by more than 8 (in units of log 2), so after the first tiles the
// sums are almost never rescaled, and the maximum over the lanes of a query is only formed when some lane needs it.  With 16-bit operands
// the sum of the probabilities comes from the matrix pipe too (a row of ones), of the values that multiply v.
#include "attention.h"

namespace lidiff {

struct AtFwd {
    const void* q;
    int64_t q_row, q_head;                                    // strides in elements
    AtRows k, v;
    const int4 *cq, *ck;                                      // (batch, x, y, z) of every row, for the biases
    const int32_t *seg_q, *seg_k;
    int nseg, mq, mk, heads, share, dim;                      // share: query heads per key head
    float scale;
    AtBias bias;
    int splits;                                               // the keys of a scan are shared out over `splits` workgroups
    void* out;                                                // [mq][heads][dim]
    float* out32;                                             // the same unrounded (for the backward pass), or null
    int exact;                                                // 16-bit operands: probabilities in pieces
    float* lse;                                               // [2][heads][mq]: log2 of the sum of exponentials in two numbers, +inf and 0 for a row without keys; or null
    float *part_o, *part_ml;                                  // splits > 1: [splits][mq][heads][dim], [splits][2][heads][mq]
};

__device__ __forceinline__ void at_put_lse(const AtFwd& a, int head, int qi, float base, float sum, float lift) {
    float rest;
    const float lse = at_two_sum(base, log2f(sum) - lift, rest);
    const bool none = sum == 0.f;
    a.lse[(int64_t)head * a.mq + qi] = none ? INFINITY : lse;
    a.lse[(int64_t)(a.heads + head) * a.mq + qi] = none ? 0.f : rest;
}

// What a workgroup takes: QB x 16 queries a wave, HG heads, tiles of 64 keys.
// HG: the distances of a (query, key) pair are the same for every head, so a wave takes as many heads as its registers hold.
// What bounds it: issue of vector instructions (41 157 x 5 824 x 2, bf16, 4 heads of 32 a wave, slopes: 1.15 ms; some 115 a head and 64 keys,
// 82 % of the cycles busy; matrix pipe 21 %, LDS 40 %).  With 16-bit operands the probabilities are rounded to their type before they meet the
// values: the output is off by 1.3 times its own rounding.  In two pieces it would be off by that rounding alone, but a training call of that
// size takes 5.08 ms then, not 4.51.  The next head's products started ahead of this head's probabilities gave nothing (1.19 against 1.18 ms;
// with the table 2.0 against 1.5: a wave less): the other waves of the SIMD fill those cycles already.
// One buffer per tile: three workgroups of a compute unit cover each other's waits better than two with a second buffer do (41 157 x 5 824
// x 2, bf16: 1.23 against 1.48 ms).  fp32 operands are three times the LDS reads: two blocks of queries share them (0.38 against 0.42 ms
// at 5 824 x 5 824; bf16: 1.41 against 1.23, for the registers).
template <typename T, int DP> struct AtFwdPlan {
    static constexpr int kHeads = sizeof(T) == 4 ? (DP == 32 ? 2 : 1) : DP == 32 ? 4 : DP == 64 ? 2 : 1;
    static constexpr int kExactHeads = kHeads > 2 ? 2 : kHeads;      // (the pieces take the registers of two heads: 1.63 against 1.91 ms at 2 x 12 809^2)
    static constexpr int kQB = sizeof(T) == 4 && DP <= 64 ? 2 : 1;
};
constexpr int kFwdRows = 64;

inline int at_fwd_heads(int most, int heads, int share, int mode) {      // whole groups of one key head, or key heads of their own
    return mode != kNone && heads % most == 0 && (share == 1 || share % most == 0) ? most : 1;
}

// EXACT (16-bit operands): probabilities enter the product with the values in pieces, rounding and rests: two where the keys are few, for the
// table's gradient as many as carry 22 to 24 bits (bf16 three, fp16 two).  d table sums ds over millions of pairs whose rows cancel to zero
// through delta = do . out, so the rounding of the probabilities behind out shows in it.  Of 2 x 12 809^2 pairs, bf16, against 64 bits: one
// piece 10^-3, two 1.2e-6, three 0.8e-6, the same in fp32 torch operations 0.8e-6; two pieces take 1.67 ms, three 2.0.
template <typename T, int DP, int HG, int SLOTS, int BIAS, int QB, bool EXACT>
__global__ __launch_bounds__(kAtBlock, at_waves(sizeof(T), DP)) void at_fwd_kernel(const AtFwd a) {
    constexpr int ROWS = kFwdRows, DC = DP / 32, DB = DP / 16, KB = ROWS / 16;
    typedef AtTile<T, DP, SLOTS, ROWS> Tile;
    typedef typename AtType<T>::Frag Frag;
    // (7, not 15: a probability may exceed the base's by 2^8)
    constexpr float kLift = AtType<T>::kLift ? 7.f : 0.f, kUnlift = AtType<T>::kLift ? 1.f / 128.f : 1.f, kSlack = 8.f;
    constexpr bool kOnes = sizeof(T) == 2 && !EXACT, kTwoLevels = sizeof(T) == 4 || EXACT;
    extern __shared__ __align__(16) char at_sm[];
    char* const ks = at_sm;
    char* const vs = ks + Tile::kBytes;
    float* const cs = reinterpret_cast<float*>(vs + Tile::kBytes);                // [2][x, y, z] of the tile's keys
    unsigned* const cells = reinterpret_cast<unsigned*>(cs + 2 * 3 * ROWS);
    float* const table = reinterpret_cast<float*>(cells + (BIAS == kTable ? kCells : 0));      // [HG][kTableRow]
    const unsigned ks_at = (unsigned)(uintptr_t)(at_lds_t)ks, vs_at = (unsigned)(uintptr_t)(at_lds_t)vs;

    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int groups = a.heads / HG, h0 = (blockIdx.x % groups) * HG, kv0 = h0 / a.share, split = blockIdx.y;
    const SegTile t = find_seg_tile(a.seg_q, a.nseg, a.mq, 64 * QB, blockIdx.x / groups);
    if (t.lo >= t.hi) return;
    const int2 kr = t.seg >= 0 ? seg_range(a.seg_k, t.seg, a.mk) : make_int2(0, 0);
    const int k_lo = __builtin_amdgcn_readfirstlane(kr.x), k_hi = __builtin_amdgcn_readfirstlane(kr.y), tiles = (k_hi - k_lo + ROWS - 1) / ROWS;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int q0 = t.lo + wave * 16 * QB;
    const float scale2 = a.scale * kLog2e;

    Frag qf[QB][HG][DC];
    float qx[QB], qy[QB], qz[QB], slope[HG];
#pragma unroll
    for (int n = 0; n < QB; ++n) {
        const int qi = q0 + 16 * n + col;
        const bool have = qi < t.hi;
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const int d = 32 * c + 8 * g;
                qf[n][h][c] = Frag{};
                if (have && d < a.dim) qf[n][h][c] = at_load8((const T*)a.q + (int64_t)qi * a.q_row + (int64_t)(h0 + h) * a.q_head + d);
            }
        qx[n] = qy[n] = qz[n] = 0.f;
        if (BIAS != kNone && have) {
            const int4 c = a.cq[qi];
            qx[n] = (float)c.y; qy[n] = (float)c.z; qz[n] = (float)c.w;
        }
    }
#pragma unroll
    for (int h = 0; h < HG; ++h) slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] / a.scale : 0.f;
    if (BIAS == kTable) {
        at_put_table<HG>(table, a.bias, a.heads, h0, a.scale);
        at_put_cells(cells, a.bias.cells);
    }

    f32x4 o[QB][HG][DB], l[QB][HG];
    float base[QB][HG];                                        // in units of log 2; -inf: nothing seen yet
    bool huge[QB][HG];
#pragma unroll
    for (int n = 0; n < QB; ++n)
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            base[n][h] = -INFINITY;
            huge[n][h] = false;
            l[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < DB; ++b) o[n][h][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    Frag ones{};
    if constexpr (kOnes) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = (typename AtType<T>::Elem)1.f;
    }

    int4 kc = make_int4(0, 0, 0, 0);                           // the coordinates one tile further than the requests
    auto coords = [&](int tile) {
        const int row = k_lo + tile * ROWS + (int)threadIdx.x;
        if (BIAS != kNone && tile < last && threadIdx.x < ROWS && row < k_hi) kc = a.ck[row];
    };
    auto put_coords = [&](int tile) {
        if (BIAS == kNone || threadIdx.x >= ROWS) return;
        float* c = cs + (tile & 1) * 3 * ROWS + threadIdx.x;
        c[0] = (float)kc.y; c[ROWS] = (float)kc.z; c[2 * ROWS] = (float)kc.w;
    };
    const char *k_at = a.k.p + (int64_t)(k_lo + first * ROWS) * a.k.row + kv0 * a.k.head, *v_at = a.v.p + (int64_t)(k_lo + first * ROWS) * a.v.row + kv0 * a.v.head;
    auto request = [&](int tile) {                             // (tile after tile)
        const int left = min(ROWS, k_hi - (k_lo + tile * ROWS));
        Tile::request(a.k, k_at, a.dim, left, ks_at);
        Tile::request(a.v, v_at, a.dim, left, vs_at);
        k_at += ROWS * a.k.row;
        v_at += ROWS * a.v.row;
    };
    const typename Tile::Lane place;
    if (first < last) {
        coords(first);
        put_coords(first);
        coords(first + 1);
        request(first);
    }
    for (int tile = first; tile < last; ++tile) {
        AT_ARRIVE();
        if (tile + 1 < last) {
            put_coords(tile + 1);
            coords(tile + 2);
        }
        if (q0 < t.hi) {                                       // (a wave without queries only takes part in the requests)
            const float* const ct = cs + (tile & 1) * 3 * ROWS;
            const int left = k_hi - (k_lo + tile * ROWS);      // keys of this tile, 64 except at the end
            AtPairs<BIAS> pairs[QB][KB];
            if (BIAS != kNone) {
#pragma unroll
                for (int n = 0; n < QB; ++n)
#pragma unroll
                    for (int b = 0; b < KB; ++b) pairs[n][b].form(ct, ROWS, 16 * b + 4 * g, qx[n], qy[n], qz[n], cells);
            }
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                const int slot = SLOTS == 1 ? 0 : h;
                f32x4 s[QB][KB];
#pragma unroll
                for (int b = 0; b < KB; ++b) {
#pragma unroll
                    for (int n = 0; n < QB; ++n) s[n][b] = pairs[n][b].start(slope[h], table, h);
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const Frag kf = Tile::frag(ks, place, slot, b, c);
#pragma unroll
                        for (int n = 0; n < QB; ++n) at_mma(s[n][b], kf, qf[n][h][c]);
                    }
                }
                if (left < ROWS) {
                    const int end = at_here(left);
#pragma unroll
                    for (int n = 0; n < QB; ++n)
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (16 * b + 4 * g + e >= end) s[n][b][e] = -INFINITY;
                            at_here(s[n][b]);
                        }
                }
                constexpr int PIECES = !EXACT ? 1 : BIAS == kTable ? AtType<T>::kPieces : 2;
                Frag p[QB][KB / 2][PIECES];
#pragma unroll
                for (int n = 0; n < QB; ++n) {
                    float top = -INFINITY;
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[n][b][e]);
                    top *= scale2;
                    if (__any(top > base[n][h] + kSlack)) {
                        top = fmaxf(top, __shfl_xor(top, 16));
                        top = fmaxf(top, __shfl_xor(top, 32));
                        const float now = fmaxf(base[n][h], top), fade = __builtin_amdgcn_exp2f(base[n][h] - (now == -INFINITY ? 0.f : now));
                        base[n][h] = now;
                        huge[n][h] = at_huge(now);
                        l[n][h] *= fade;
#pragma unroll
                        for (int b = 0; b < DB; ++b) o[n][h][b] *= fade;
                    }
                    float down = base[n][h] == -INFINITY ? 0.f : kLift - base[n][h], factor = scale2;
                    if (huge[n][h]) {                          // (the lift would be lost beside such a base as well)
                        const float f = __builtin_bit_cast(float, at_here(__builtin_bit_cast(int, scale2))), from = base[n][h] == -INFINITY ? 0.f : base[n][h];
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[n][b][e] = at_exponent(s[n][b][e], f, from);
                            at_here(s[n][b]);
                        }
                        factor = 1.f;
                        down = kLift;
                    }
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[n][b][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[n][b][e], factor, down));
                            if (!kOnes) l[n][h][e] += s[n][b][e];
                        }
#pragma unroll
                    for (int j = 0; j < KB / 2; ++j) {
                        f32x8 v = at_join(s[n][2 * j], s[n][2 * j + 1]);
                        at_pack(p[n][j][0], v);
                        if constexpr (PIECES > 1) {
#pragma unroll
                            for (int i = 1; i < PIECES; ++i) at_pack_rest(p[n][j][i], p[n][j][i - 1], v);
                        }
                        if constexpr (kOnes) {
#pragma unroll
                            for (int i = 0; i < PIECES; ++i) at_mma(l[n][h], ones, p[n][j][i]);
                        }
                    }
                }
                // (kTwoLevels: the matrix pipe rounds a long chain of sums to one side; where fp32 is asked for, a tile is summed by itself)
                f32x4 part[QB][DB];
#pragma unroll
                for (int n = 0; n < QB; ++n)
#pragma unroll
                    for (int b = 0; b < DB; ++b) part[n][b] = kTwoLevels ? f32x4{0.f, 0.f, 0.f, 0.f} : o[n][h][b];
#pragma unroll
                for (int j = 0; j < KB / 2; ++j)
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        const Frag vf = Tile::frag_turned(vs, place, slot, j, b);
#pragma unroll
                        for (int n = 0; n < QB; ++n)
#pragma unroll
                            for (int i = 0; i < PIECES; ++i) at_mma(part[n][b], vf, p[n][j][i]);
                    }
#pragma unroll
                for (int n = 0; n < QB; ++n)
#pragma unroll
                    for (int b = 0; b < DB; ++b) o[n][h][b] = kTwoLevels ? o[n][h][b] + part[n][b] : part[n][b];
            }
        }
        if (tile + 1 < last) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");        // the tile has been read
            request(tile + 1);
        }
    }
#pragma unroll
    for (int n = 0; n < QB; ++n) {
        const int qi = q0 + 16 * n + col;
        if (qi >= t.hi) continue;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            float sum = l[n][h][0];                            // (ones: every row of the product holds the sum)
            if (!kOnes) {
                sum = (l[n][h][0] + l[n][h][1]) + (l[n][h][2] + l[n][h][3]);
                sum += __shfl_xor(sum, 16);                    // (the four lanes of a query are here together)
                sum += __shfl_xor(sum, 32);
            }
            const int head = h0 + h;
            if (a.splits > 1) {
                if (g == 0) {
                    a.part_ml[((int64_t)(2 * split) * a.heads + head) * a.mq + qi] = base[n][h];
                    a.part_ml[((int64_t)(2 * split + 1) * a.heads + head) * a.mq + qi] = sum * kUnlift;
                }
#pragma unroll
                for (int b = 0; b < DB; ++b)
                    if (16 * b + 4 * g < a.dim) at_store4(a.part_o + (((int64_t)split * a.mq + qi) * a.heads + head) * a.dim + 16 * b + 4 * g, o[n][h][b] * kUnlift);
                continue;
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (a.lse && g == 0) at_put_lse(a, head, qi, base[n][h], sum, kLift);
#pragma unroll
            for (int b = 0; b < DB; ++b) {
                if (16 * b + 4 * g >= a.dim) continue;
                const f32x4 r = o[n][h][b] * inv;
                const int64_t at = ((int64_t)qi * a.heads + head) * a.dim + 16 * b + 4 * g;
                at_store4((T*)a.out + at, r);
                if (a.out32) at_store4(a.out32 + at, r);
            }
        }
    }
}

// Joins the shares of the keys.  A (query, head) takes `width` lanes of four elements, times `lanes` that each add every lanes-th share; a
// fixed butterfly joins those.  Many shares are read side by side (one lane walking over 45 of them: 23 us against 6), few by one lane
// each (3 shares of 46 592 units: 7 us against 19).
template <typename T>
__global__ __launch_bounds__(256) void at_join_kernel(const AtFwd a, int width, int lanes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, unit = i / (width * lanes);
    if (unit >= (int64_t)a.mq * a.heads) return;              // (units are whole groups of lanes: a butterfly stays inside one)
    const int head = (int)(unit % a.heads), qi = (int)(unit / a.heads), d = (int)(i % width) * 4, first = (int)(i / width % lanes);
    const float* const ml = a.part_ml + (int64_t)head * a.mq + qi;
    const int64_t plane = (int64_t)a.heads * a.mq;
    float m = -INFINITY;
    for (int s = first; s < a.splits; s += lanes) m = fmaxf(m, ml[2 * s * plane]);
    for (int off = width * lanes / 2; off >= width; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = first; s < a.splits; s += lanes) {
        const float w = __builtin_amdgcn_exp2f(ml[2 * s * plane] - base);
        sum += w * ml[(2 * s + 1) * plane];
        if (d < a.dim) o += w * *reinterpret_cast<const f32x4*>(a.part_o + (((int64_t)s * a.mq + qi) * a.heads + head) * a.dim + d);
    }
    for (int off = width * lanes / 2; off >= width; off >>= 1) {
        sum += __shfl_xor(sum, off);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off);
    }
    if (a.lse && d == 0 && first == 0) at_put_lse(a, head, qi, m, sum, 0.f);
    if (first != 0 || d >= a.dim) return;
    const f32x4 r = o * (sum == 0.f ? 0.f : 1.f / sum);
    const int64_t at = ((int64_t)qi * a.heads + head) * a.dim + d;
    at_store4((T*)a.out + at, r);
    if (a.out32) at_store4(a.out32 + at, r);
}

template <typename T, int DP, int HG, int SLOTS, int BIAS, bool EXACT>
static hipError_t at_fwd_launch(const AtFwd& a, hipStream_t st) {
    typedef AtFwdPlan<T, DP> Plan;
    constexpr int QB = Plan::kQB;
    const int64_t wg = seg_tiles_bound(a.mq, 64 * QB, a.seg_q, a.nseg) * (a.heads / HG);
    size_t lds = (size_t)2 * AtTile<T, DP, SLOTS, kFwdRows>::kBytes + 2 * 3 * kFwdRows * sizeof(float);
    if (BIAS == kTable) lds += (kCells + kTableRow * HG) * sizeof(float);
    auto kern = at_fwd_kernel<T, DP, HG, SLOTS, BIAS, QB, EXACT>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    kern<<<dim3((unsigned)wg, (unsigned)a.splits), kAtBlock, lds, st>>>(a);
    if (a.splits > 1) {
        const int width = DP / 4, lanes = a.splits > 8 ? kWave / width : 1;
        at_join_kernel<T><<<(unsigned)ceil_div((int64_t)a.mq * a.heads * width * lanes, 256), 256, 0, st>>>(a, width, lanes);
    }
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS, bool EXACT = false>
static hipError_t at_fwd_bias(const AtFwd& a, int mode, hipStream_t st) {
    if (mode == kTable) return at_fwd_launch<T, DP, HG, SLOTS, kTable, EXACT>(a, st);
    if (mode == kSlope) return at_fwd_launch<T, DP, HG, SLOTS, kSlope, EXACT>(a, st);
    if constexpr (HG == 1) return at_fwd_launch<T, DP, HG, SLOTS, kNone, EXACT>(a, st);
    return hipErrorInvalidValue;
}

template <typename T, int DP>
static hipError_t at_fwd_width(const AtFwd& a, int mode, hipStream_t st) {
    constexpr int most = AtFwdPlan<T, DP>::kHeads, exact = AtFwdPlan<T, DP>::kExactHeads;
    if constexpr (sizeof(T) == 2) {
        if (a.exact) {
            if constexpr (exact > 1)
                if (at_fwd_heads(exact, a.heads, a.share, mode) == exact)
                    return a.share > 1 ? at_fwd_bias<T, DP, exact, 1, true>(a, mode, st) : at_fwd_bias<T, DP, exact, exact, true>(a, mode, st);
            return at_fwd_bias<T, DP, 1, 1, true>(a, mode, st);
        }
    }
    if constexpr (most > 1)
        if (at_fwd_heads(most, a.heads, a.share, mode) == most) return a.share > 1 ? at_fwd_bias<T, DP, most, 1>(a, mode, st) : at_fwd_bias<T, DP, most, most>(a, mode, st);
    return at_fwd_bias<T, DP, 1, 1>(a, mode, st);
}

// how many workgroups share a scan's keys: one while there are workgroups enough for the card, else so many that there are, each with
// at least two tiles of an average scan's keys
template <typename T, int DP>
static int at_fwd_splits(int64_t mq, int64_t mk, int64_t nseg, int heads, int share, int mode) {
    typedef AtFwdPlan<T, DP> Plan;
    const int64_t wg = (ceil_div(mq, 64 * Plan::kQB) + nseg - 1) * (heads / at_fwd_heads(Plan::kHeads, heads, share, mode));
    if (wg >= 512) return 1;
    const int64_t want = ceil_div(1024, wg), most = ceil_div(mk, nseg) / (2 * kFwdRows);
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : (int)(n < 64 ? n : 64);
}

struct AtFwdLayout { int splits; int64_t k, v, part, bytes; };      // workspace: the planes of k and v (fp32), the shares' sums

template <typename T>
static AtFwdLayout at_fwd_layout(int64_t mq, int64_t mk, int64_t nseg, int heads, int kv_heads, int dim, int mode) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    AtFwdLayout l;
    const int share = heads / kv_heads;
    l.splits = dim <= 32 ? at_fwd_splits<T, 32>(mq, mk, nseg, heads, share, mode) : dim <= 64 ? at_fwd_splits<T, 64>(mq, mk, nseg, heads, share, mode)
                                                                                            : at_fwd_splits<T, 128>(mq, mk, nseg, heads, share, mode);
    const int64_t planes = sizeof(T) == 4 ? up(3 * at_plane_bytes(mk, kv_heads, dim)) : 0;
    l.k = 0;
    l.v = planes;
    l.part = 2 * planes;
    l.bytes = l.part + (l.splits > 1 ? l.splits * mq * heads * (dim + 2) * (int64_t)sizeof(float) : 0);
    return l;
}

struct AtFwdIn {
    const void *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    int kv_heads;
    char* ws;
};

template <typename T>
static hipError_t at_fwd_run(AtFwd a, const AtFwdIn& in, const AtFwdLayout& l, int mode, hipStream_t st) {
    a.k = at_stream<T>(in.k, in.k_row, in.k_head, a.mk, in.kv_heads, a.dim, in.ws + l.k, st);
    a.v = at_stream<T>(in.v, in.v_row, in.v_head, a.mk, in.kv_heads, a.dim, in.ws + l.v, st);
    if (a.dim <= 32) return at_fwd_width<T, 32>(a, mode, st);
    if (a.dim <= 64) return at_fwd_width<T, 64>(a, mode, st);
    return at_fwd_width<T, 128>(a, mode, st);
}

}  // namespace lidiff

using namespace lidiff;

static AtFwdLayout at_fwd_layout_of(int dtype, int64_t mq, int64_t mk, int64_t nseg, int heads, int kv_heads, int dim, int mode) {
    return dtype == 0 ? at_fwd_layout<float>(mq, mk, nseg, heads, kv_heads, dim, mode) : at_fwd_layout<__bf16>(mq, mk, nseg, heads, kv_heads, dim, mode);
}

extern "C" int64_t lidiff_segment_attention_workspace_bytes(int64_t mq, int64_t mk, int64_t n_segments, int32_t heads, int32_t kv_heads, int32_t dim,
                                                            int32_t dtype, int32_t bias_mode) {
    if (mq < 1 || mk < 0 || n_segments < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 128) return 0;
    return at_fwd_layout_of(dtype, mq, mk, n_segments, heads, kv_heads, dim, bias_mode).bytes;
}

extern "C" int lidiff_segment_attention(const void* q, const void* k, const void* v, const int64_t* strides, const int32_t* coords_q, const int32_t* coords_k,
                                        const int32_t* seg_q, const int32_t* seg_k, int64_t n_segments, int64_t mq, int64_t mk, int32_t heads,
                                        int32_t kv_heads, int32_t dim, int32_t dtype, float scale, int32_t bias_mode, const float* slopes,
                                        const float* table, const void* cells, int32_t buckets, void* out, float* out_f32, int32_t exact, float* lse,
                                        void* workspace, void* stream) {
    LIDIFF_CHECK_ARG(q && out && strides && (mk == 0 || (k && v)), "null pointer");
    const char* bad = at_check(n_segments, mq, mk, heads, kv_heads, dim, dtype, scale, bias_mode, buckets, strides, 6);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG((seg_q != nullptr) == (seg_k != nullptr) && (seg_q || n_segments == 1), "segments of queries and keys come together");
    LIDIFF_CHECK_ARG(bias_mode == kNone || (coords_q && (coords_k || mk == 0)), "a distance bias needs the coordinates");
    LIDIFF_CHECK_ARG(bias_mode != kSlope || slopes, "null pointer");
    LIDIFF_CHECK_ARG(bias_mode != kTable || (table && cells), "null pointer");
    LIDIFF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)out_f32 | (uintptr_t)coords_q | (uintptr_t)coords_k |
                       (uintptr_t)workspace) & 15) == 0 && (((uintptr_t)seg_q | (uintptr_t)seg_k) & 7) == 0, "misaligned pointer");
    const AtFwdLayout l = at_fwd_layout_of(dtype, mq, mk, n_segments, heads, kv_heads, dim, bias_mode);
    LIDIFF_CHECK_ARG(l.bytes == 0 || workspace, "workspace missing (lidiff_segment_attention_workspace_bytes)");
    AtFwd a;
    a.q = q; a.q_row = strides[0]; a.q_head = strides[1];
    a.cq = (const int4*)coords_q; a.ck = (const int4*)coords_k;
    a.seg_q = seg_q; a.seg_k = seg_k; a.nseg = (int)n_segments; a.mq = (int)mq; a.mk = (int)mk;
    a.heads = heads; a.share = heads / kv_heads; a.dim = dim;
    a.scale = scale;
    a.bias = AtBias{table, (const unsigned*)cells, slopes, bias_mode == kTable ? buckets : 0};
    a.splits = l.splits;
    a.out = out; a.out32 = out_f32; a.exact = exact; a.lse = lse;
    a.part_o = (float*)((char*)workspace + l.part);
    a.part_ml = a.part_o + (int64_t)l.splits * mq * heads * dim;
    const AtFwdIn in = {k, v, strides[2], strides[3], strides[4], strides[5], kv_heads, (char*)workspace};
    hipStream_t st = (hipStream_t)stream;
    LIDIFF_CHECK_HIP(dtype == 0 ? at_fwd_run<float>(a, in, l, bias_mode, st) : dtype == 1 ? at_fwd_run<__bf16>(a, in, l, bias_mode, st)
                                                                                          : at_fwd_run<_Float16>(a, in, l, bias_mode, st));
    return 0;
}
