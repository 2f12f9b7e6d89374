// Attention between the rows of the same scan, backward.  With s = q . k scale + bias, p = exp(s - lse) (rebuilt from the forward pass's
// sums), delta_i = sum_d do_i out_i and ds = p (do . v - delta):
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i,   d table[b][h] = sum of ds over the pairs of bucket b.
// What bounds them: issue of vector instructions, then LDS (41 157 x 5 824 x 2, 8 heads of 32, bf16, slopes: dq 1.23 ms, dk / dv 1.80 ms =
// 0.58 and 0.53 PFLOP/s of their three and four products; vector issue 81 and 72 %, LDS 54 and 65 %, matrix pipe 24 and 22 % of the cycles).
// fp32 operands: neither pipe is full (7 702 x 5 824 x 2, 4 heads of 64, table: vector 52 %, matrix 33 and 40 %): 1.8 waves a SIMD wait a
// third of their time.
// 16-bit operands: probabilities and score gradients are rounded once, to the operands' type, before their products: gradients are off by
// 1.4 to 1.6 times their own rounding (the last where few keys share a row and delta carries the output's rounded probabilities).
// Two kernels that each own their outputs (queries; keys), so nothing is added by atomics and every run gives the same bits: seven products
// per pair and channel instead of five.  delta and the gradient of the table take the UNROUNDED output of the forward pass: the rows of ds
// sum to zero only as exactly as delta is known.
//
// fp16 operands.  A score gradient is a probability times a gradient and soon lies below fp16's range (2^-24), so it is multiplied by a
// power of two before it is rounded and the sums are multiplied back, both exact.  Every sum (a query's dq, a key's dk) has a power of its
// own that follows its largest score gradient so far, as a softmax's running maximum does (at_lift_to): no other row, of this scan or of
// another, moves it.
#include "attention.h"

namespace lidiff {

struct AtBwd {
    const void *q, *k, *v, *go;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, go_row, go_head;      // strides in elements
    AtRows qs, ks, vs, gs;                                    // the same tensors as they are streamed
    const int4 *cq, *ck;
    const int32_t *seg_q, *seg_k;
    int nseg, mq, mk, heads, share, dim;
    float scale;
    AtBias bias;
    const float *out32, *lse;                                 // [mq][heads][dim], [2][heads][mq]
    float* stat;                                              // [3][heads][mq]: lse (less kLift), -delta, lse's second number, for the dk / dv kernel
    void *dq, *dk, *dv;                                       // contiguous
    int splits;                                               // dk / dv: the queries of a scan are shared out over `splits` workgroups
    float* part_kv;                                           // splits > 1: [splits][2][mk][heads / share][dim]
    float* part_t;                                            // [tiles][heads][buckets]
    int tiles;
};

// Multiplies a column's score gradients (its four lanes hold 4 N each) by the column's power of two `lift`; where the largest would leave
// [0, 2^15] the power is lowered so that it comes to [2^10, 2^11) -- 2^4 of room for the next tiles' -- and the sums formed so far go along.
// 2^-24 of the largest keeps all of fp16's bits, and what fp16 loses below is 2^-34 of it.  Values that are not finite make their sum so
// and leave the power alone.
constexpr float kLiftStart = 1152921504606846976.f;          // 2^60: within fp32 times the largest |ds| (2^41, with p's own lift 2^56), beyond 2^15 times any that matters
template <int N, int DB>
__device__ __forceinline__ void at_lift_to(float& lift, f32x4 (&ds)[N], f32x4 (&sums)[DB]) {
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(ds[b][e]));
    if (__any(top * lift > 32768.f)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int was = __builtin_bit_cast(int, lift) >> 23, most = 127 + 10 - ((__builtin_bit_cast(int, top) >> 23) - 127);
        const bool lower = top * lift > 32768.f && top < INFINITY;
        const float fade = __builtin_bit_cast(float, (lower ? most - was + 127 : 127) << 23);
        lift *= fade;
#pragma unroll
        for (int b = 0; b < DB; ++b) sums[b] *= fade;
    }
#pragma unroll
    for (int b = 0; b < N; ++b) ds[b] *= lift;
}
__device__ __forceinline__ float at_unlift(float lift) { return __builtin_bit_cast(float, (254 << 23) - __builtin_bit_cast(int, lift)); }      // 1 / 2^n, exact

// (At 2 heads of 32 with the table's gradient, 16-bit: 74 to 82 registers of the 256 are spilled, of dk / dv 2 to 11.)
// What a workgroup takes: heads at a time (the distances of a pair are the same for every head), rows of a tile.  One buffer per tile, as in
// the forward kernel (41 157 x 5 824 x 2, bf16, dq: 1.43 against 1.69 ms).
template <typename T, int DP> struct AtBwdPlan {
    static constexpr int kHeads = sizeof(T) == 4 ? (DP == 32 ? 2 : 1) : DP == 32 ? 4 : DP == 64 ? 2 : 1;
    static constexpr int kKeyHeads = kHeads > 2 ? 2 : kHeads;         // dk / dv: twice the accumulators (four waves a SIMD: 1.56 against 1.71 ms)
    static constexpr int kGradHeads = sizeof(T) == 4 ? 1 : DP == 32 ? 2 : 1;      // with the table's gradient: a histogram of 256 bytes a wave, bucket and head
    static constexpr int kGradRows = 32;
    static constexpr int kGradQB = sizeof(T) == 2 && DP == 32 ? 2 : 1;      // blocks of 16 queries a wave (2.58 against 2.81 ms; fp32: 1.14 against 0.97)
    static constexpr int kRows = 64, kQB = 1;                         // (two blocks: 1.33 against 1.26 ms)
    // dk / dv, 128 wide: three waves with four registers spilled against two without, 949 : 995 us at 20 000 x 5 824, bf16, slopes, 2 heads, training
    static constexpr int kKeyWaves = sizeof(T) == 2 ? (DP == 32 ? 4 : DP == 128 ? 3 : 2) : at_waves(sizeof(T), DP);
};

inline int at_bwd_heads(int most, int heads, int share, int mode) {      // whole groups of one key head, or key heads of their own
    return mode != kNone && heads % most == 0 && (share == 1 || share % most == 0) ? most : 1;
}

// Adds the score gradients of four pairs and HG heads to the words of a lane's own column, [bucket][HG][64 lanes] (place: byte offsets
// of a row of the table, four per bucket).  LDS float atomics take some 240 cycles a wave (15.9 ms of the gradient of 3 10^8
// pairs x 8 heads); plain reads and writes of a private column need no atomic.  A wave's accesses happen in order: two pairs at a time, for
// all heads, are read and written; if their buckets are the same the second, written last, holds both.
template <int HG>
__device__ __forceinline__ void at_hist(char* __restrict__ column, const int (&place)[4], const f32x4 (&v)[HG]) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        float* const one = reinterpret_cast<float*>(column + place[e] * (64 * HG));
        float* const two = reinterpret_cast<float*>(column + place[e + 1] * (64 * HG));
        const bool same = place[e] == place[e + 1];
        float a[HG], b[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) { a[h] = one[h * 64]; b[h] = two[h * 64]; }
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            a[h] += v[h][e];
            b[h] = (same ? a[h] : b[h]) + v[h][e + 1];
        }
#pragma unroll
        for (int h = 0; h < HG; ++h) one[h * 64] = a[h];
#pragma unroll
        for (int h = 0; h < HG; ++h) two[h * 64] = b[h];
    }
}

// one workgroup: 64 QB queries of one scan x HG heads: dq, delta, and its part of the table's gradient
template <typename T, int DP, int HG, int SLOTS, int BIAS, bool GRAD, int ROWS, int QB>
__global__ __launch_bounds__(kAtBlock, at_waves(sizeof(T), DP)) void at_bwd_q_kernel(const AtBwd a) {
    constexpr int DC = DP / 32, DB = DP / 16;
    typedef AtTile<T, DP, SLOTS, ROWS> Tile;
    typedef typename AtType<T>::Frag Frag;
    constexpr bool kLifted = AtType<T>::kLift != 0;
    extern __shared__ __align__(16) char at_sm[];
    char* const ks = at_sm;
    char* const vs = ks + Tile::kBytes;
    float* const cs = reinterpret_cast<float*>(vs + Tile::kBytes);
    unsigned* const cells = reinterpret_cast<unsigned*>(cs + 2 * 3 * ROWS);
    float* const table = reinterpret_cast<float*>(cells + (BIAS == kTable ? kCells : 0));
    float* const hist = table + (BIAS == kTable ? kTableRow * HG : 0);              // [wave][bucket][HG][64 lanes]: a lane adds to words of its own
    const unsigned ks_at = (unsigned)(uintptr_t)(at_lds_t)ks, vs_at = (unsigned)(uintptr_t)(at_lds_t)vs;

    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int groups = a.heads / HG, h0 = (blockIdx.x % groups) * HG, kv0 = h0 / a.share, tile_id = blockIdx.x / groups;
    const SegTile t = find_seg_tile(a.seg_q, a.nseg, a.mq, 64 * QB, tile_id);
    if (t.lo >= t.hi) {
        if (GRAD)
            for (int i = threadIdx.x; i < HG * a.bias.buckets; i += kAtBlock)
                a.part_t[((int64_t)tile_id * a.heads + h0) * a.bias.buckets + i] = 0.f;
        return;
    }
    const int2 kr = t.seg >= 0 ? seg_range(a.seg_k, t.seg, a.mk) : make_int2(0, 0);
    const int k_lo = __builtin_amdgcn_readfirstlane(kr.x), k_hi = __builtin_amdgcn_readfirstlane(kr.y);
    // (one key: its probability is 1 whatever its score is, so there are no score gradients -- do . v less do . out would be their roundings)
    const int last = k_hi - k_lo == 1 ? 0 : (k_hi - k_lo + ROWS - 1) / ROWS;
    const int q0 = t.lo + wave * 16 * QB;
    const float scale2 = a.scale * kLog2e;

    Frag qf[QB][HG][DC], gf[QB][HG][DC];
    float lse[QB][HG], slope[HG], lift[QB][HG], qx[QB], qy[QB], qz[QB];
    bool far[QB][HG];
    // -delta: what the products do . v start from.  (With the table's gradient it is added behind them: the matrix pipe rounds sums to one
    // side, and what is the same for every pair does not cancel in a sum over 10^8 of them -- 1.9e-5 of the gradient against 1.2e-6.)
    float less[QB][HG];
    // That side is the lower one also within one product (of fp16's 22 bits more than of bf16's 16 are cut): with do turned for every other
    // query the cuts fall to both sides alike, for no instruction more (fp16,
    // 15 158 x 3 082 pairs of 96: 1.2e-6 of the gradient against 1.3e-5; times as before).
    const float sign = GRAD && (col & 1) ? -1.f : 1.f;
#pragma unroll
    for (int n = 0; n < QB; ++n) {
        const int qi = q0 + 16 * n + col;
        const bool have = qi < t.hi;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const int d = 32 * c + 8 * g;
                qf[n][h][c] = gf[n][h][c] = Frag{};
                if (have && d < a.dim) {
                    const T* go = (const T*)a.go + (int64_t)qi * a.go_row + (int64_t)(h0 + h) * a.go_head + d;
                    qf[n][h][c] = at_load8((const T*)a.q + (int64_t)qi * a.q_row + (int64_t)(h0 + h) * a.q_head + d);
                    gf[n][h][c] = at_load8(go);
                    if (GRAD) at_turn(gf[n][h][c], col & 1 ? 0x80008000u : 0u);
                    const float* o = a.out32 + ((int64_t)qi * a.heads + h0 + h) * a.dim + d;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += (float)go[e] * o[e];
                }
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            less[n][h] = -sum;
            lse[n][h] = have ? a.lse[(int64_t)(h0 + h) * a.mq + qi] : INFINITY;
            if (have && g == 0) {
                float off;                                     // (the lift may not move lse's last bits either)
                a.stat[(int64_t)(h0 + h) * a.mq + qi] = at_two_sum(lse[n][h], -(float)AtType<T>::kLift, off);
                a.stat[(int64_t)(a.heads + h0 + h) * a.mq + qi] = -sum;
                a.stat[(int64_t)(2 * a.heads + h0 + h) * a.mq + qi] = a.lse[(int64_t)(a.heads + h0 + h) * a.mq + qi] + off;
            }
            lift[n][h] = kLiftStart;
            far[n][h] = at_far(lse[n][h]);
        }
        qx[n] = qy[n] = qz[n] = 0.f;
        if (BIAS != kNone) {                                   // (a place without a query stands where the last one does: it meets no bucket that
            const int4 c = a.cq[min(qi, t.hi - 1)];            // no query meets, whose entry may be infinite or NaN)
            qx[n] = (float)c.y; qy[n] = (float)c.z; qz[n] = (float)c.w;
        }
    }
#pragma unroll
    for (int h = 0; h < HG; ++h) slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] / a.scale : 0.f;
    if (BIAS == kTable) {
        at_put_table<HG>(table, a.bias, a.heads, h0, a.scale);
        at_put_cells(cells, a.bias.cells);
        if (GRAD)
            for (int i = threadIdx.x; i < 4 * a.bias.buckets * HG * 64; i += kAtBlock) hist[i] = 0.f;
    }
    char* const mine = reinterpret_cast<char*>(hist + wave * a.bias.buckets * HG * 64 + lane);

    f32x4 dq[QB][HG][DB];
#pragma unroll
    for (int n = 0; n < QB; ++n)
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int b = 0; b < DB; ++b) dq[n][h][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The columns' sums go over into doubles every kGather tiles: a word then holds a few hundred values, and its rounding does not show in
    // the sum of 3 10^8 (5 10^-7 of it with 2 000 a word).
    constexpr int kGather = 64, kSums = (4 * HG * 48 + kAtBlock - 1) / kAtBlock;
    double sums[kSums] = {};
    auto gather = [&]() {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            const int i = k * kAtBlock + threadIdx.x;
            if (i >= 4 * HG * a.bias.buckets) continue;
            double u = 0;                                      // (64 lanes in a fixed order; neighbouring threads in neighbouring banks)
            for (int l = 0; l < 64; ++l) {
                float& word = hist[i * 64 + ((l + i) & 63)];
                u += word;
                word = 0.f;
            }
            sums[k] += u;
        }
        __syncthreads();
    };

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
    const char *k_at = a.ks.p + (int64_t)k_lo * a.ks.row + kv0 * a.ks.head, *v_at = a.vs.p + (int64_t)k_lo * a.vs.row + kv0 * a.vs.head;
    auto request = [&](int tile) {                             // (tile after tile)
        const int left = min(ROWS, k_hi - (k_lo + tile * ROWS));
        Tile::request(a.ks, k_at, a.dim, left, ks_at);
        Tile::request(a.vs, v_at, a.dim, left, vs_at);
        k_at += ROWS * a.ks.row;
        v_at += ROWS * a.vs.row;
    };
    const typename Tile::Lane place;
    if (last > 0) {
        coords(0);
        put_coords(0);
        coords(1);
        request(0);
    }
    for (int tile = 0; tile < last; ++tile) {
        AT_ARRIVE();
        if (tile + 1 < last) {
            put_coords(tile + 1);
            coords(tile + 2);
        }
        if (q0 < t.hi) {
            const float* const ct = cs + (tile & 1) * 3 * ROWS;
            const int left = k_hi - (k_lo + tile * ROWS);
#pragma unroll
            for (int j = 0; j < ROWS / 32; ++j) {              // 32 keys at a time
                AtPairs<BIAS> pairs[QB][2];
                f32x4 grads[QB][2][HG];
                if (BIAS != kNone) {
#pragma unroll
                    for (int n = 0; n < QB; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b) pairs[n][b].form(ct, ROWS, 32 * j + 16 * b + 4 * g, qx[n], qy[n], qz[n], cells);
                }
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    const int slot = SLOTS == 1 ? 0 : h;
                    f32x4 s[QB][2], dp[QB][2];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
#pragma unroll
                        for (int n = 0; n < QB; ++n) {
                            s[n][b] = pairs[n][b].start(slope[h], table, h);
                            dp[n][b] = GRAD ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{less[n][h], less[n][h], less[n][h], less[n][h]};
                        }
#pragma unroll
                        for (int c = 0; c < DC; ++c) {
                            const Frag kf = Tile::frag(ks, place, slot, 2 * j + b, c), vf = Tile::frag(vs, place, slot, 2 * j + b, c);
#pragma unroll
                            for (int n = 0; n < QB; ++n) {
                                at_mma(s[n][b], kf, qf[n][h][c]);
                                if (GRAD) at_mma_apart(dp[n][b], vf, gf[n][h][c]);
                                else at_mma(dp[n][b], vf, gf[n][h][c]);
                            }
                        }
                    }
                    Frag p[QB];
#pragma unroll
                    for (int n = 0; n < QB; ++n) {
                        float factor = scale2, minus = lse[n][h];
                        if (far[n][h]) {                       // (lse's second number from memory: the branch is rare, registers are not spent on it)
                            const float f = __builtin_bit_cast(float, at_here(__builtin_bit_cast(int, scale2)));
                            const float rest = a.lse[(int64_t)(a.heads + h0 + h) * a.mq + min(at_here(q0 + 16 * n + col), t.hi - 1)];
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[n][b][e] = at_exponent(s[n][b][e], f, lse[n][h]) - rest;
                                at_here(s[n][b]);
                            }
                            factor = 1.f;
                            minus = 0.f;
                        }
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[n][b][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[n][b][e], factor, -minus));
#pragma unroll
                        for (int b = 0; b < 2; ++b) s[n][b] *= GRAD ? dp[n][b] * sign + less[n][h] : dp[n][b];
                        if (left < ROWS) {
                            const int end = at_here(left);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (32 * j + 16 * b + 4 * g + e >= end) s[n][b][e] = 0.f;
                                at_here(s[n][b]);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < 2; ++b)
                            if (GRAD) grads[n][b][h] = s[n][b];
                        if constexpr (kLifted) at_lift_to(lift[n][h], s[n], dq[n][h]);
                        at_pack(p[n], at_join(s[n][0], s[n][1]));
                    }
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        const Frag kf = Tile::frag_turned(ks, place, slot, j, b);
#pragma unroll
                        for (int n = 0; n < QB; ++n) at_mma_rows(dq[n][h][b], kf, p[n]);
                    }
                }
                if (GRAD) {
#pragma unroll
                    for (int n = 0; n < QB; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b) at_hist<HG>(mine, pairs[n][b].b, grads[n][b]);
                }
            }
        }
        if (GRAD && (tile + 1) % kGather == 0) gather();       // (every wave is here)
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
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int b = 0; b < DB; ++b)
                if (16 * b + 4 * g < a.dim)
                    at_store4((T*)a.dq + ((int64_t)qi * a.heads + h0 + h) * a.dim + 16 * b + 4 * g, dq[n][h][b] * (kLifted ? a.scale * at_unlift(lift[n][h]) : a.scale));
    }
    if (GRAD) {
        gather();
        double* const wide = reinterpret_cast<double*>(hist);
#pragma unroll
        for (int k = 0; k < kSums; ++k)
            if (k * kAtBlock + threadIdx.x < 4 * HG * a.bias.buckets) wide[k * kAtBlock + threadIdx.x] = sums[k];
        __syncthreads();
        for (int i = threadIdx.x; i < HG * a.bias.buckets; i += kAtBlock) {
            double u = 0;
            for (int w = 0; w < 4; ++w) u += wide[w * HG * a.bias.buckets + i];
            a.part_t[((int64_t)tile_id * a.heads + h0 + i % HG) * a.bias.buckets + i / HG] = (float)u;
        }
    }
}

// one workgroup: 64 keys of one scan x SLOTS key heads x one share of the queries: dk, dv
template <typename T, int DP, int HG, int SLOTS, int BIAS>
__global__ __launch_bounds__(kAtBlock, (AtBwdPlan<T, DP>::kKeyWaves)) void at_bwd_kv_kernel(const AtBwd a) {
    constexpr int ROWS = 64, DC = DP / 32, DB = DP / 16;
    typedef AtTile<T, DP, HG, ROWS> Tile;
    typedef typename AtType<T>::Frag Frag;
    constexpr bool kLifted = AtType<T>::kLift != 0;
    extern __shared__ __align__(16) char at_sm[];
    char* const qs = at_sm;
    char* const gs = qs + Tile::kBytes;
    float* const st = reinterpret_cast<float*>(gs + Tile::kBytes);                 // [2][HG][64] lse, -delta
    float* const cs = st + 2 * HG * ROWS;
    unsigned* const cells = reinterpret_cast<unsigned*>(cs + 2 * 3 * ROWS);
    float* const table = reinterpret_cast<float*>(cells + (BIAS == kTable ? kCells : 0));
    const unsigned qs_at = (unsigned)(uintptr_t)(at_lds_t)qs, gs_at = (unsigned)(uintptr_t)(at_lds_t)gs, st_at = (unsigned)(uintptr_t)(at_lds_t)st;

    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int kv_heads = a.heads / a.share, groups = kv_heads / SLOTS, kv0 = (blockIdx.x % groups) * SLOTS, split = blockIdx.y;
    const SegTile t = find_seg_tile(a.seg_k, a.nseg, a.mk, 64, blockIdx.x / groups);
    if (t.lo >= t.hi) return;
    const int2 qr = t.seg >= 0 ? seg_range(a.seg_q, t.seg, a.mq) : make_int2(0, 0);
    const int q_lo = __builtin_amdgcn_readfirstlane(qr.x), q_hi = __builtin_amdgcn_readfirstlane(qr.y), tiles = (q_hi - q_lo + ROWS - 1) / ROWS;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int k0 = t.lo + wave * 16, ki = k0 + col;
    const bool have = ki < t.hi;
    const float scale2 = a.scale * kLog2e;

    Frag kf[SLOTS][DC], vf[SLOTS][DC];
    float lift[SLOTS];
    f32x4 dk[SLOTS][DB], dv[SLOTS][DB];
#pragma unroll
    for (int h = 0; h < SLOTS; ++h) {
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = 32 * c + 8 * g;
            kf[h][c] = vf[h][c] = Frag{};
            if (have && d < a.dim) {
                kf[h][c] = at_load8((const T*)a.k + (int64_t)ki * a.k_row + (int64_t)(kv0 + h) * a.k_head + d);
                vf[h][c] = at_load8((const T*)a.v + (int64_t)ki * a.v_row + (int64_t)(kv0 + h) * a.v_head + d);
            }
        }
        lift[h] = kLiftStart;
#pragma unroll
        for (int b = 0; b < DB; ++b) dk[h][b] = dv[h][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr float kUnlift = kLifted ? 1.f / (1 << AtType<T>::kLift) : 1.f;
    float kx = 0.f, ky = 0.f, kz = 0.f;
    if (BIAS != kNone && have) {
        const int4 c = a.ck[ki];
        kx = (float)c.y; ky = (float)c.z; kz = (float)c.w;
    }
    if (BIAS == kTable)
        at_put_cells(cells, a.bias.cells);

    const typename Tile::Lane place;
    // the query heads that read these key heads, HG at a time
    for (int h0 = kv0 * a.share; h0 < (kv0 + SLOTS) * a.share; h0 += HG) {
        float slope[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] / a.scale : 0.f;
        int4 qc = make_int4(0, 0, 0, 0);
        auto coords = [&](int tile) {
            const int row = q_lo + tile * ROWS + (int)threadIdx.x;
            if (BIAS != kNone && tile < last && threadIdx.x < ROWS && row < q_hi) qc = a.cq[row];
        };
        auto put_coords = [&](int tile) {
            if (BIAS == kNone || threadIdx.x >= ROWS) return;
            float* c = cs + (tile & 1) * 3 * ROWS + threadIdx.x;
            c[0] = (float)qc.y; c[ROWS] = (float)qc.z; c[2 * ROWS] = (float)qc.w;
        };
        const char *q_at = a.qs.p + (int64_t)(q_lo + first * ROWS) * a.qs.row + h0 * a.qs.head, *g_at = a.gs.p + (int64_t)(q_lo + first * ROWS) * a.gs.row + h0 * a.gs.head;
        auto request = [&](int tile) {                         // (tile after tile)
            const int lo = q_lo + tile * ROWS, left = min(ROWS, q_hi - lo);
            Tile::request(a.qs, q_at, a.dim, left, qs_at);
            Tile::request(a.gs, g_at, a.dim, left, gs_at);
            q_at += ROWS * a.qs.row;
            g_at += ROWS * a.gs.row;
            for (int i = wave; i < 2 * HG; i += 4) {           // lse and -delta: 64 words a head
                const uint64_t base = (uint64_t)(uintptr_t)(a.stat + ((int64_t)(i / HG) * a.heads + h0 + i % HG) * a.mq + lo);
                i32x4 rsrc = {(int)(uint32_t)base, (int)(uint32_t)((base >> 32) & 0xffffu), left * 4, 0x00020000};
#pragma unroll
                for (int k = 0; k < 4; ++k) rsrc[k] = __builtin_amdgcn_readfirstlane(rsrc[k]);
                lds_dma4(rsrc, __builtin_amdgcn_readfirstlane(st_at + i * ROWS * 4), lane * 4, 0);
            }
        };
        __syncthreads();                                       // the chunk of heads before has been read
        if (BIAS == kTable) at_put_table<HG>(table, a.bias, a.heads, h0, a.scale);
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
            if (k0 < t.hi) {
                bool far[HG];
#pragma unroll
                for (int h = 0; h < HG; ++h) far[h] = at_far(st[h * ROWS + lane]);
                const float* const ct = cs + (tile & 1) * 3 * ROWS;
                const int left = q_hi - (q_lo + tile * ROWS);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    AtPairs<BIAS> pairs[2];
                    if (BIAS != kNone) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) pairs[b].form(ct, ROWS, 32 * j + 16 * b + 4 * g, kx, ky, kz, cells);
                    }
#pragma unroll
                    for (int h = 0; h < HG; ++h) {
                        const int slot = SLOTS == 1 ? 0 : h;
                        f32x4 s[2], dp[2];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const f32x4 lse = *reinterpret_cast<const f32x4*>(st + h * ROWS + 32 * j + 16 * b + 4 * g);
                            s[b] = pairs[b].start(slope[h], table, h);
                            dp[b] = *reinterpret_cast<const f32x4*>(st + (HG + h) * ROWS + 32 * j + 16 * b + 4 * g);
#pragma unroll
                            for (int c = 0; c < DC; ++c) {
                                at_mma(s[b], Tile::frag(qs, place, h, 2 * j + b, c), kf[slot][c]);
                                at_mma(dp[b], Tile::frag(gs, place, h, 2 * j + b, c), vf[slot][c]);
                            }
                            if (far[h]) {                      // (lse's second numbers from memory, as above)
                                const float f = __builtin_bit_cast(float, at_here(__builtin_bit_cast(int, scale2)));
                                const float* const rest = a.stat + (int64_t)(2 * a.heads + h0 + h) * a.mq;
                                const int row = at_here(q_lo + tile * ROWS + 32 * j + 16 * b + 4 * g);
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[b][e] = __builtin_amdgcn_exp2f(at_exponent(s[b][e], f, lse[e]) - rest[min(row + e, q_hi - 1)]);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[b][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[b][e], scale2, -lse[e]));
                            }
                        }
                        if (left < ROWS) {
                            const int end = at_here(left);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (32 * j + 16 * b + 4 * g + e >= end) s[b][e] = 0.f;
                                at_here(s[b]);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < 2; ++b) dp[b] *= s[b];
                        if constexpr (kLifted) at_lift_to(lift[slot], dp, dk[slot]);
                        Frag p, ds;
                        at_pack(p, at_join(s[0], s[1]));
                        at_pack(ds, at_join(dp[0], dp[1]));
#pragma unroll
                        for (int b = 0; b < DB; ++b) {
                            at_mma_rows(dv[slot][b], Tile::frag_turned(gs, place, h, j, b), p);
                            at_mma_rows(dk[slot][b], Tile::frag_turned(qs, place, h, j, b), ds);
                        }
                    }
                }
            }
            if (tile + 1 < last) {
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                request(tile + 1);
            }
        }
    }
    if (!have) return;
    if (t.hi - t.lo == 1 && t.seg >= 0) {                      // (a lone key has no score gradients, as above)
        const int2 own = seg_range(a.seg_k, t.seg, a.mk);
        if (own.y - own.x == 1)
#pragma unroll
            for (int h = 0; h < SLOTS; ++h)
#pragma unroll
                for (int b = 0; b < DB; ++b) dk[h][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int h = 0; h < SLOTS; ++h) {
        // (p, and with it ds, carries kLift already)
        const float dk_unlift = kLifted ? at_unlift(lift[h]) * kUnlift : 1.f;
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            if (16 * b + 4 * g >= a.dim) continue;
            const int64_t at = ((int64_t)ki * kv_heads + kv0 + h) * a.dim + 16 * b + 4 * g;
            if (a.splits > 1) {
                const int64_t plane = (int64_t)a.mk * kv_heads * a.dim;
                at_store4(a.part_kv + (2 * split) * plane + at, dk[h][b] * dk_unlift);
                at_store4(a.part_kv + (2 * split + 1) * plane + at, dv[h][b] * kUnlift);
            } else {
                at_store4((T*)a.dk + at, dk[h][b] * (a.scale * dk_unlift));
                at_store4((T*)a.dv + at, dv[h][b] * kUnlift);
            }
        }
    }
}

template <typename T>
__global__ void at_join_kv_kernel(const AtBwd a) {
    const int64_t plane = (int64_t)a.mk * (a.heads / a.share) * a.dim, i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (i >= plane) return;
    f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
    for (int s = 0; s < a.splits; ++s) {
        dk += *reinterpret_cast<const f32x4*>(a.part_kv + (2 * s) * plane + i);
        dv += *reinterpret_cast<const f32x4*>(a.part_kv + (2 * s + 1) * plane + i);
    }
    at_store4((T*)a.dk + i, dk * a.scale);
    at_store4((T*)a.dv + i, dv);
}

// d table[b][h]: one wave adds the workgroups' parts in a fixed order
__global__ __launch_bounds__(kWave) void at_table_kernel(const float* __restrict__ part, int tiles, int heads, int buckets, float* __restrict__ out) {
    const int b = blockIdx.x / heads, h = blockIdx.x % heads;
    double u = 0;
    for (int t = threadIdx.x; t < tiles; t += kWave) u += part[((int64_t)t * heads + h) * buckets + b];
    for (int off = kWave / 2; off > 0; off >>= 1) u += __shfl_down(u, off);
    if (threadIdx.x == 0) out[(int64_t)b * heads + h] = (float)u;
}

template <typename T, int DP, int HG, int SLOTS, int BIAS, bool GRAD>
static hipError_t at_bwd_q_launch(const AtBwd& a, hipStream_t st) {
    typedef AtBwdPlan<T, DP> Plan;
    constexpr int ROWS = GRAD ? Plan::kGradRows : Plan::kRows, QB = GRAD ? Plan::kGradQB : Plan::kQB;
    size_t lds = (size_t)2 * AtTile<T, DP, SLOTS, ROWS>::kBytes + 2 * 3 * ROWS * sizeof(float);
    if (BIAS == kTable) lds += (kCells + kTableRow * HG) * sizeof(float);
    if (GRAD) lds += (size_t)4 * a.bias.buckets * HG * 64 * sizeof(float);
    auto kern = at_bwd_q_kernel<T, DP, HG, SLOTS, BIAS, GRAD, ROWS, QB>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    kern<<<(unsigned)(seg_tiles_bound(a.mq, 64 * QB, a.seg_q, a.nseg) * (a.heads / HG)), kAtBlock, lds, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS, int BIAS>
static hipError_t at_bwd_kv_launch(const AtBwd& a, hipStream_t st) {
    size_t lds = (size_t)2 * AtTile<T, DP, HG, 64>::kBytes + (2 * HG + 2 * 3) * 64 * sizeof(float);
    if (BIAS == kTable) lds += (kCells + kTableRow * HG) * sizeof(float);
    auto kern = at_bwd_kv_kernel<T, DP, HG, SLOTS, BIAS>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    const int64_t wg = seg_tiles_bound(a.mk, 64, a.seg_k, a.nseg) * (a.heads / a.share / SLOTS);
    kern<<<dim3((unsigned)wg, (unsigned)a.splits), kAtBlock, lds, st>>>(a);
    if (a.splits > 1)
        at_join_kv_kernel<T><<<(unsigned)ceil_div((int64_t)a.mk * (a.heads / a.share) * a.dim / 4, 256), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS>
static hipError_t at_bwd_q_bias(const AtBwd& a, int mode, hipStream_t st) {
    if (mode == kTable) return at_bwd_q_launch<T, DP, HG, SLOTS, kTable, false>(a, st);
    if (mode == kSlope) return at_bwd_q_launch<T, DP, HG, SLOTS, kSlope, false>(a, st);
    if constexpr (HG == 1) return at_bwd_q_launch<T, DP, HG, SLOTS, kNone, false>(a, st);
    return hipErrorInvalidValue;
}

template <typename T, int DP, int HG, int SLOTS>
static hipError_t at_bwd_kv_bias(const AtBwd& a, int mode, hipStream_t st) {
    if (mode == kTable) return at_bwd_kv_launch<T, DP, HG, SLOTS, kTable>(a, st);
    if (mode == kSlope) return at_bwd_kv_launch<T, DP, HG, SLOTS, kSlope>(a, st);
    if constexpr (HG == 1) return at_bwd_kv_launch<T, DP, HG, SLOTS, kNone>(a, st);
    return hipErrorInvalidValue;
}

template <typename T, int DP>
static hipError_t at_bwd_width(const AtBwd& a, int mode, hipStream_t st) {
    constexpr int most = AtBwdPlan<T, DP>::kHeads, grad = AtBwdPlan<T, DP>::kGradHeads, keys = AtBwdPlan<T, DP>::kKeyHeads;
    const bool wide = most > 1 && at_bwd_heads(most, a.heads, a.share, mode) == most, one = a.share > 1;
    hipError_t e;
    if (a.part_t) {
        e = hipErrorInvalidValue;
        if constexpr (grad > 1) {
            if (at_bwd_heads(grad, a.heads, a.share, mode) == grad)
                e = one ? at_bwd_q_launch<T, DP, grad, 1, kTable, true>(a, st) : at_bwd_q_launch<T, DP, grad, grad, kTable, true>(a, st);
            else e = at_bwd_q_launch<T, DP, 1, 1, kTable, true>(a, st);
        } else e = at_bwd_q_launch<T, DP, 1, 1, kTable, true>(a, st);
    } else if (wide) e = one ? at_bwd_q_bias<T, DP, most, 1>(a, mode, st) : at_bwd_q_bias<T, DP, most, most>(a, mode, st);
    else e = at_bwd_q_bias<T, DP, 1, 1>(a, mode, st);
    if (e != hipSuccess || a.dk == nullptr) return e;
    if (keys > 1 && at_bwd_heads(keys, a.heads, a.share, mode) == keys) return one ? at_bwd_kv_bias<T, DP, keys, 1>(a, mode, st) : at_bwd_kv_bias<T, DP, keys, keys>(a, mode, st);
    return at_bwd_kv_bias<T, DP, 1, 1>(a, mode, st);
}

// Shares of the queries for dk / dv: so many that there are two workgroups of a compute unit each and the last round of them is not a
// large part of the time, each with at least two tiles of an average scan's queries.
template <typename T, int DP>
static int at_bwd_splits(int64_t mq, int64_t mk, int64_t nseg, int heads, int kv_heads, int mode) {
    const int share = heads / kv_heads, slots = share > 1 ? 1 : at_bwd_heads(AtBwdPlan<T, DP>::kKeyHeads, heads, share, mode);
    const int64_t wg = (ceil_div(mk > 0 ? mk : 1, 64) + nseg - 1) * (kv_heads / slots);
    if (wg >= 2048) return 1;
    const int64_t want = ceil_div(2048, wg), most = ceil_div(mq, nseg) / 128;
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : (int)(n < 64 ? n : 64);
}

inline int at_grad_blocks(int dtype, int dim) {
    return dtype == 0 ? (dim <= 32 ? AtBwdPlan<float, 32>::kGradQB : dim <= 64 ? AtBwdPlan<float, 64>::kGradQB : AtBwdPlan<float, 128>::kGradQB)
                      : (dim <= 32 ? AtBwdPlan<__bf16, 32>::kGradQB : dim <= 64 ? AtBwdPlan<__bf16, 64>::kGradQB : AtBwdPlan<__bf16, 128>::kGradQB);
}

struct AtBwdLayout { int splits; int64_t q, k, v, go, table, kv, bytes; };      // workspace; the row statistics come first

template <typename T>
static AtBwdLayout at_bwd_layout(int64_t mq, int64_t mk, const void* seg, int64_t nseg, int heads, int kv_heads, int dim, int mode, int buckets, bool table_grad) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    AtBwdLayout l;
    l.splits = dim <= 32 ? at_bwd_splits<T, 32>(mq, mk, nseg, heads, kv_heads, mode) : dim <= 64 ? at_bwd_splits<T, 64>(mq, mk, nseg, heads, kv_heads, mode)
                                                                                               : at_bwd_splits<T, 128>(mq, mk, nseg, heads, kv_heads, mode);
    const int64_t pq = sizeof(T) == 4 ? up(3 * at_plane_bytes(mq, heads, dim)) : 0, pk = sizeof(T) == 4 ? up(3 * at_plane_bytes(mk, kv_heads, dim)) : 0;
    l.q = up(3 * mq * heads * (int64_t)sizeof(float));
    l.go = l.q + pq;
    l.k = l.go + pq;
    l.v = l.k + pk;
    l.table = l.v + pk;
    l.kv = l.table + (table_grad ? up(seg_tiles_bound(mq, 64, seg, nseg) * heads * buckets * (int64_t)sizeof(float)) : 0);
    l.bytes = l.kv + (l.splits > 1 ? up(2 * l.splits * mk * kv_heads * dim * (int64_t)sizeof(float)) : 0);
    return l;
}

template <typename T>
static hipError_t at_bwd_run(AtBwd a, const AtBwdLayout& l, int mode, char* ws, hipStream_t st) {
    const int kv_heads = a.heads / a.share;
    a.ks = at_stream<T>(a.k, a.k_row, a.k_head, a.mk, kv_heads, a.dim, ws + l.k, st);
    a.vs = at_stream<T>(a.v, a.v_row, a.v_head, a.mk, kv_heads, a.dim, ws + l.v, st);
    if (a.dk) {
        a.qs = at_stream<T>(a.q, a.q_row, a.q_head, a.mq, a.heads, a.dim, ws + l.q, st);
        a.gs = at_stream<T>(a.go, a.go_row, a.go_head, a.mq, a.heads, a.dim, ws + l.go, st);
    }
    if (a.dim <= 32) return at_bwd_width<T, 32>(a, mode, st);
    if (a.dim <= 64) return at_bwd_width<T, 64>(a, mode, st);
    return at_bwd_width<T, 128>(a, mode, st);
}

static AtBwdLayout at_bwd_layout_of(int dtype, int64_t mq, int64_t mk, const void* seg, int64_t nseg, int heads, int kv_heads, int dim, int mode, int buckets,
                                    bool table_grad) {
    return dtype == 0 ? at_bwd_layout<float>(mq, mk, seg, nseg, heads, kv_heads, dim, mode, buckets, table_grad)
                      : at_bwd_layout<__bf16>(mq, mk, seg, nseg, heads, kv_heads, dim, mode, buckets, table_grad);
}

}  // namespace lidiff

using namespace lidiff;

extern "C" int64_t lidiff_segment_attention_bwd_workspace_bytes(int64_t mq, int64_t mk, int64_t n_segments, int32_t heads, int32_t kv_heads, int32_t dim,
                                                                int32_t dtype, int32_t bias_mode, int32_t buckets, int32_t table_grad) {
    if (mq < 1 || mk < 0 || n_segments < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 128) return 0;
    return at_bwd_layout_of(dtype, mq, mk, &mq, n_segments, heads, kv_heads, dim, bias_mode, buckets, table_grad != 0).bytes;      // (with segments: the larger bound)
}

extern "C" int lidiff_segment_attention_bwd(const void* q, const void* k, const void* v, const void* grad_out, const int64_t* strides,
                                            const int32_t* coords_q, const int32_t* coords_k, const int32_t* seg_q, const int32_t* seg_k,
                                            int64_t n_segments, int64_t mq, int64_t mk, int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype,
                                            float scale, int32_t bias_mode, const float* slopes, const float* table, const void* cells, int32_t buckets,
                                            const float* out_f32, const float* lse, void* dq, void* dk, void* dv, float* dtable, void* workspace,
                                            void* stream) {
    LIDIFF_CHECK_ARG(q && grad_out && strides && out_f32 && lse && dq && workspace && (mk == 0 || (k && v)) && (dk != nullptr) == (dv != nullptr), "null pointer");
    const char* bad = at_check(n_segments, mq, mk, heads, kv_heads, dim, dtype, scale, bias_mode, buckets, strides, 8);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG((seg_q != nullptr) == (seg_k != nullptr) && (seg_q || n_segments == 1), "segments of queries and keys come together");
    LIDIFF_CHECK_ARG(bias_mode == kNone || (coords_q && (coords_k || mk == 0)), "a distance bias needs the coordinates");
    LIDIFF_CHECK_ARG(bias_mode != kSlope || slopes, "null pointer");
    LIDIFF_CHECK_ARG(bias_mode != kTable || (table && cells), "null pointer");
    LIDIFF_CHECK_ARG(dtable == nullptr || bias_mode == kTable, "a table gradient without a table");
    LIDIFF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)grad_out | (uintptr_t)out_f32 | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv |
                       (uintptr_t)coords_q | (uintptr_t)coords_k | (uintptr_t)workspace) & 15) == 0 &&
                     (((uintptr_t)seg_q | (uintptr_t)seg_k) & 7) == 0, "misaligned pointer");
    AtBwd a;
    a.q = q; a.k = k; a.v = v; a.go = grad_out;
    a.q_row = strides[0]; a.q_head = strides[1]; a.k_row = strides[2]; a.k_head = strides[3]; a.v_row = strides[4]; a.v_head = strides[5];
    a.go_row = strides[6]; a.go_head = strides[7];
    a.cq = (const int4*)coords_q; a.ck = (const int4*)coords_k;
    a.seg_q = seg_q; a.seg_k = seg_k; a.nseg = (int)n_segments; a.mq = (int)mq; a.mk = (int)mk;
    a.heads = heads; a.share = heads / kv_heads; a.dim = dim;
    a.scale = scale;
    a.bias = AtBias{table, (const unsigned*)cells, slopes, bias_mode == kTable ? buckets : 0};
    a.out32 = out_f32; a.lse = lse;
    a.dq = dq; a.dk = mk > 0 ? dk : nullptr; a.dv = dv;
    const AtBwdLayout l = at_bwd_layout_of(dtype, mq, mk, seg_q, n_segments, heads, kv_heads, dim, bias_mode, buckets, dtable != nullptr);
    char* ws = (char*)workspace;
    a.stat = (float*)ws;
    a.part_t = dtable ? (float*)(ws + l.table) : nullptr;
    a.part_kv = (float*)(ws + l.kv);
    a.tiles = (int)seg_tiles_bound(mq, 64 * at_grad_blocks(dtype, dim), seg_q, n_segments);
    a.splits = l.splits;
    hipStream_t st = (hipStream_t)stream;
    LIDIFF_CHECK_HIP(dtype == 0 ? at_bwd_run<float>(a, l, bias_mode, ws, st) : dtype == 1 ? at_bwd_run<__bf16>(a, l, bias_mode, ws, st)
                                                                                        : at_bwd_run<_Float16>(a, l, bias_mode, ws, st));
    if (dtable) {
        at_table_kernel<<<(unsigned)(buckets * heads), kWave, 0, st>>>(a.part_t, a.tiles, heads, buckets, dtable);
        LIDIFF_CHECK_LAUNCH();
    }
    return 0;
}
