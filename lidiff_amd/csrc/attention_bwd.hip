// Attention between the rows of the same scan, backward.  With s = q . k scale + bias, p = exp(s - lse) (rebuilt from the forward pass's
// sums), delta_i = sum_d do_i out_i and ds = p (do . v - delta):
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i,   d table[b][h] = sum of ds over the pairs of bucket b.
// Two kernels that each own their outputs (queries; keys), so nothing is added by atomics and every run gives the same bits: seven products
// per pair and channel instead of five.  delta and the gradient of the table take the UNROUNDED output of the forward pass: the rows of ds
// sum to zero only as exactly as delta is known.
//
// fp16 operands.  A score gradient is a probability times a gradient and soon lies below fp16's range (2^-24), so it is multiplied by a
// power of two before it is rounded and the sums are multiplied back, both exact: |ds| <= 2 |do_i| max_j |v_j|, and the power takes that
// bound to 2^15.  dq: a power of each query; dk: one for all queries of a key head (a sum has one scale).  The norms' maxima come from a
// pass of their own over do and v; values that are not finite take no part in them.
#include "attention.h"

namespace lidiff {

struct AtBwd {
    const void *q, *k, *v, *go;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, go_row, go_head;
    const int4 *cq, *ck;
    const int32_t *seg_q, *seg_k;
    int nseg, mq, mk, heads, share, dim;
    float scale;                                              // as it is (not times log2 e)
    AtBias bias;
    const float *out32, *lse;                                 // [mq][heads][dim], [heads][mq]
    float* delta;                                             // [heads][mq]
    void *dq, *dk, *dv;                                       // contiguous
    int splits;                                               // dk / dv: the queries of a scan are shared out over `splits` workgroups
    float* part_kv;                                           // splits > 1: [splits][2][mk][heads / share][dim]
    float* part_t;                                            // [tiles][heads][buckets]
    int tiles;
    unsigned* bound;                                          // fp16: [2][heads / share] bits of the largest |do|^2 and |v|^2 of a key head
};

// the power of two (its exponent) for score gradients bounded by 2 sqrt(g2 v2)
__device__ __forceinline__ float at_lift(float g2, float v2) {
    return fminf(fmaxf(floorf(14.f - 0.5f * (__builtin_amdgcn_logf(g2) + __builtin_amdgcn_logf(v2))), -100.f), 100.f);
}

__global__ void at_bound_clear_kernel(unsigned* bound, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) bound[i] = 0u;
}

// largest |row|^2 of a head of src [rows][heads][dim], joined over `share` heads: a maximum of bit patterns, the same in any order
template <typename T>
__global__ __launch_bounds__(256) void at_bound_kernel(const T* __restrict__ src, int64_t row_stride, int64_t head_stride, int rows, int dim, int share,
                                                      unsigned* __restrict__ bound) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    float sum = 0.f;
    if (row < rows) {
        const T* p = src + row * row_stride + (int64_t)blockIdx.y * head_stride;
        for (int d = 0; d < dim; ++d) sum += (float)p[d] * (float)p[d];
    }
    if (!(sum < INFINITY)) sum = 0.f;
    for (int off = kWave / 2; off > 0; off >>= 1) sum = fmaxf(sum, __shfl_xor(sum, off));
    if (lane_id() == 0) atomicMax(bound + blockIdx.y / share, __builtin_bit_cast(unsigned, sum));
}

// one workgroup: 64 queries of one scan x HG heads: dq, delta, and its part of the table's gradient
template <typename T, int DP, int HG, int SLOTS, int BIAS, bool GRAD>
__global__ __launch_bounds__(kAtBlock) void at_bwd_q_kernel(const AtBwd a) {
    typedef AtTile<T, DP> Tile;
    typedef typename AtType<T>::Frag Frag;
    constexpr int DC = DP / 32, DB = DP / 16;
    constexpr bool kLifted = AtType<T>::kLift != 0;
    extern __shared__ __align__(16) unsigned char at_sm[];
    T* ks = reinterpret_cast<T*>(at_sm);
    T* vs = ks + SLOTS * Tile::kRows;
    T* kt = vs + SLOTS * Tile::kRows;
    float* cs = reinterpret_cast<float*>(kt + SLOTS * Tile::kCols);
    float* table = cs + 3 * kAtRows;
    AtCell* cells = reinterpret_cast<AtCell*>(table + (BIAS == kTable ? ((a.bias.buckets * HG + 3) & ~3) : 0));
    float* hist = reinterpret_cast<float*>(cells + (BIAS == kTable ? kCells : 0));      // [wave][bucket][HG][64 lanes]: a lane adds to its own word only

    const int lane = lane_id(), wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const int groups = a.heads / HG, h0 = (blockIdx.x % groups) * HG, kv0 = h0 / a.share, tile_id = blockIdx.x / groups;
    const SegTile t = find_seg_tile(a.seg_q, a.nseg, a.mq, kAtRows, tile_id);
    if (t.lo >= t.hi) {
        if (GRAD)
            for (int i = threadIdx.x; i < HG * a.bias.buckets; i += kAtBlock)
                a.part_t[((int64_t)tile_id * a.heads + h0 + i / a.bias.buckets) * a.bias.buckets + i % a.bias.buckets] = 0.f;
        return;
    }
    const int qi = t.lo + wave * 16 + col;
    const bool have = qi < t.hi;
    const int2 kr = t.seg >= 0 ? seg_range(a.seg_k, t.seg, a.mk) : make_int2(0, 0);
    const int tiles = (kr.y - kr.x + kAtRows - 1) / kAtRows;
    const float scale2 = a.scale * kLog2e;

    Frag qf[HG][DC], gf[HG][DC];
    float lse[HG], delta[HG], slope[HG], unlift[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
        float sum = 0.f, g2 = 0.f;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = 32 * c + 8 * g;
            const bool in = have && d < a.dim;
            qf[h][c] = in ? at_frag((const T*)a.q + (int64_t)qi * a.q_row + (int64_t)(h0 + h) * a.q_head + d) : at_zero<T>();
            const T* go = (const T*)a.go + (int64_t)qi * a.go_row + (int64_t)(h0 + h) * a.go_head + d;
            gf[h][c] = in ? at_frag(go) : at_zero<T>();
            if (in) {
                const float* o = a.out32 + ((int64_t)qi * a.heads + h0 + h) * a.dim + d;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum += (float)go[e] * o[e];
                    if (kLifted) g2 += (float)go[e] * (float)go[e];
                }
            }
        }
        sum += __shfl_xor(sum, 16);
        delta[h] = sum + __shfl_xor(sum, 32);
        lse[h] = have ? a.lse[(int64_t)(h0 + h) * a.mq + qi] : INFINITY;
        if (have && g == 0) a.delta[(int64_t)(h0 + h) * a.mq + qi] = delta[h];
        unlift[h] = 1.f;
        if (kLifted) {
            g2 += __shfl_xor(g2, 16);
            g2 += __shfl_xor(g2, 32);
            const int kv_heads = a.heads / a.share;
            const float lift = at_lift(g2, __builtin_bit_cast(float, a.bound[kv_heads + (h0 + h) / a.share]));
            lse[h] -= lift;                                    // p, and with it ds, carries the power of two
            unlift[h] = __builtin_amdgcn_exp2f(-lift);
        }
        slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] * kLog2e : 0.f;
    }
    float qx = 0.f, qy = 0.f, qz = 0.f;
    if (BIAS != kNone && have) {
        const int4 c = a.cq[qi];
        qx = (float)c.y; qy = (float)c.z; qz = (float)c.w;
    }
    if (BIAS == kTable) {
        for (int i = threadIdx.x; i < a.bias.buckets * HG; i += kAtBlock) table[i] = a.bias.table[(int64_t)(i / HG) * a.heads + h0 + i % HG] * kLog2e;
        for (int i = threadIdx.x; i < kCells; i += kAtBlock) cells[i] = a.bias.cells[i];
        if (GRAD)
            for (int i = threadIdx.x; i < 4 * a.bias.buckets * HG * 64; i += kAtBlock) hist[i] = 0.f;
    }
    float* mine = hist + (int64_t)wave * a.bias.buckets * HG * 64 + lane;

    f32x4 dq[HG][DB] = {};
    AtLoad<T, DP, SLOTS> kl, vl;
    int4 kc = make_int4(0, 0, 0, 0);
    auto fetch = [&](int tile) {
        const int lo = kr.x + tile * kAtRows;
        kl.fetch((const T*)a.k, a.k_row, a.k_head, kv0, a.dim, lo, kr.y);
        vl.fetch((const T*)a.v, a.v_row, a.v_head, kv0, a.dim, lo, kr.y);
        if (BIAS != kNone && threadIdx.x < kAtRows && lo + (int)threadIdx.x < kr.y) kc = a.ck[lo + threadIdx.x];
    };
    if (tiles > 0) fetch(0);
    for (int tile = 0; tile < tiles; ++tile) {
        __syncthreads();
        kl.put_rows(ks);
        kl.put_cols(kt);
        vl.put_rows(vs);
        if (BIAS != kNone && threadIdx.x < kAtRows) {
            cs[threadIdx.x] = (float)kc.y;
            cs[kAtRows + threadIdx.x] = (float)kc.z;
            cs[2 * kAtRows + threadIdx.x] = (float)kc.w;
        }
        __syncthreads();
        if (tile + 1 < tiles) fetch(tile + 1);
        if (t.lo + wave * 16 >= t.hi) continue;
        const int left = kr.y - (kr.x + tile * kAtRows);
#pragma unroll
        for (int j = 0; j < 2; ++j) {                          // 32 keys at a time
            float dist[8];
            int row_of[8];
            if (BIAS != kNone) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int at = 32 * j + 16 * b + 4 * g;
                    const f32x4 x = *reinterpret_cast<const f32x4*>(cs + at), y = *reinterpret_cast<const f32x4*>(cs + kAtRows + at),
                                z = *reinterpret_cast<const f32x4*>(cs + 2 * kAtRows + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float dx = x[e] - qx, dy = y[e] - qy, dz = z[e] - qz, d2 = dx * dx + dy * dy + dz * dz;
                        if (BIAS == kSlope) dist[4 * b + e] = __builtin_amdgcn_sqrtf(d2);
                        if (BIAS == kTable) {
                            const AtCell c = cells[at_cell(d2)];
                            row_of[4 * b + e] = c.bucket + (d2 >= c.edge ? 1 : 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                const int slot = SLOTS == 1 ? 0 : h;
                f32x4 s[2], dp[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
                    dp[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const int at = slot * Tile::kRows + (32 * j + 16 * b + col) * Tile::kRow + 32 * c + 8 * g;
                        at_mma(s[b], at_frag(ks + at), qf[h][c]);
                        at_mma(dp[b], at_frag(vs + at), gf[h][c]);
                    }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = s[b][e] * scale2;
                        if (BIAS == kSlope) v += slope[h] * dist[4 * b + e];
                        if (BIAS == kTable) v += table[row_of[4 * b + e] * HG + h];
                        float p = __builtin_amdgcn_exp2f(v - lse[h]);
                        if (left < kAtRows && 32 * j + 16 * b + 4 * g + e >= left) p = 0.f;
                        s[b][e] = p * (dp[b][e] - delta[h]);
                        if (GRAD) __hip_atomic_fetch_add(mine + (row_of[4 * b + e] * HG + h) * 64, s[b][e] * unlift[h], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    }
                Frag p;
                at_pack(p, s[0], s[1]);
#pragma unroll
                for (int b = 0; b < DB; ++b) at_mma(dq[h][b], at_frag_rows(kt + slot * Tile::kCols + (16 * b + col) * Tile::kCol + 32 * j + 4 * g), p);
            }
        }
    }
    if (have) {
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int b = 0; b < DB; ++b)
                if (16 * b + 4 * g < a.dim) at_store4((T*)a.dq + ((int64_t)qi * a.heads + h0 + h) * a.dim + 16 * b + 4 * g, dq[h][b] * (a.scale * unlift[h]));
    }
    if (GRAD) {
        __syncthreads();
        for (int i = threadIdx.x; i < HG * a.bias.buckets; i += kAtBlock) {
            const int b = i / HG, h = i % HG;
            double u = 0;                                      // (the 4 x 64 lanes' sums in a fixed order)
            for (int w = 0; w < 4; ++w)
                for (int l = 0; l < 64; ++l) u += hist[((w * a.bias.buckets + b) * HG + h) * 64 + ((l + i) & 63)];
            a.part_t[((int64_t)tile_id * a.heads + h0 + h) * a.bias.buckets + b] = (float)u;
        }
    }
}

// one workgroup: 64 keys of one scan x SLOTS key heads x one share of the queries: dk, dv
template <typename T, int DP, int HG, int SLOTS, int BIAS>
__global__ __launch_bounds__(kAtBlock) void at_bwd_kv_kernel(const AtBwd a) {
    typedef AtTile<T, DP> Tile;
    typedef typename AtType<T>::Frag Frag;
    constexpr int DC = DP / 32, DB = DP / 16;
    constexpr bool kLifted = AtType<T>::kLift != 0;
    extern __shared__ __align__(16) unsigned char at_sm[];
    T* qs = reinterpret_cast<T*>(at_sm);
    T* gs = qs + HG * Tile::kRows;
    T* qt = gs + HG * Tile::kRows;
    T* gt = qt + HG * Tile::kCols;
    float* cs = reinterpret_cast<float*>(gt + HG * Tile::kCols);                  // x, y, z, then [HG][64] lse, [HG][64] delta
    float* ls = cs + 3 * kAtRows;
    float* ds = ls + HG * kAtRows;
    float* table = ds + HG * kAtRows;
    AtCell* cells = reinterpret_cast<AtCell*>(table + (BIAS == kTable ? ((a.bias.buckets * HG + 3) & ~3) : 0));

    const int lane = lane_id(), wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const int kv_heads = a.heads / a.share, groups = kv_heads / SLOTS, kv0 = (blockIdx.x % groups) * SLOTS, split = blockIdx.y;
    const SegTile t = find_seg_tile(a.seg_k, a.nseg, a.mk, kAtRows, blockIdx.x / groups);
    if (t.lo >= t.hi) return;
    const int ki = t.lo + wave * 16 + col;
    const bool have = ki < t.hi;
    const int2 qr = t.seg >= 0 ? seg_range(a.seg_q, t.seg, a.mq) : make_int2(0, 0);
    const int tiles = (qr.y - qr.x + kAtRows - 1) / kAtRows;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
    const float scale2 = a.scale * kLog2e;

    Frag kf[SLOTS][DC], vf[SLOTS][DC];
#pragma unroll
    for (int h = 0; h < SLOTS; ++h)
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = 32 * c + 8 * g;
            const bool in = have && d < a.dim;
            kf[h][c] = in ? at_frag((const T*)a.k + (int64_t)ki * a.k_row + (int64_t)(kv0 + h) * a.k_head + d) : at_zero<T>();
            vf[h][c] = in ? at_frag((const T*)a.v + (int64_t)ki * a.v_row + (int64_t)(kv0 + h) * a.v_head + d) : at_zero<T>();
        }
    float kx = 0.f, ky = 0.f, kz = 0.f;
    if (BIAS != kNone && have) {
        const int4 c = a.ck[ki];
        kx = (float)c.y; ky = (float)c.z; kz = (float)c.w;
    }
    if (BIAS == kTable)
        for (int i = threadIdx.x; i < kCells; i += kAtBlock) cells[i] = a.bias.cells[i];

    float ds_lift[SLOTS], dk_unlift[SLOTS];
#pragma unroll
    for (int h = 0; h < SLOTS; ++h) {
        ds_lift[h] = dk_unlift[h] = 1.f;
        if (kLifted) {
            const float lift = at_lift(__builtin_bit_cast(float, a.bound[kv0 + h]), __builtin_bit_cast(float, a.bound[kv_heads + kv0 + h]));
            ds_lift[h] = __builtin_amdgcn_exp2f(lift - AtType<T>::kLift);             // (p carries kLift already)
            dk_unlift[h] = __builtin_amdgcn_exp2f(-lift);
        }
    }
    constexpr float kUnlift = kLifted ? 1.f / (1 << AtType<T>::kLift) : 1.f;

    f32x4 dk[SLOTS][DB] = {}, dv[SLOTS][DB] = {};
    // the query heads that read these key heads, HG at a time
    for (int h0 = kv0 * a.share; h0 < (kv0 + SLOTS) * a.share; h0 += HG) {
        AtLoad<T, DP, HG> ql, gl;
        int4 qc = make_int4(0, 0, 0, 0);
        float lse_r[(HG * kAtRows + kAtBlock - 1) / kAtBlock], delta_r[(HG * kAtRows + kAtBlock - 1) / kAtBlock], slope[HG];
        auto fetch = [&](int tile) {
            const int lo = qr.x + tile * kAtRows;
            ql.fetch((const T*)a.q, a.q_row, a.q_head, h0, a.dim, lo, qr.y);
            gl.fetch((const T*)a.go, a.go_row, a.go_head, h0, a.dim, lo, qr.y);
            if (BIAS != kNone && threadIdx.x < kAtRows && lo + (int)threadIdx.x < qr.y) qc = a.cq[lo + threadIdx.x];
#pragma unroll
            for (int p = 0; p < (HG * kAtRows + kAtBlock - 1) / kAtBlock; ++p) {
                const int i = p * kAtBlock + threadIdx.x, row = lo + i % kAtRows;
                const bool in = i < HG * kAtRows && row < qr.y;
                lse_r[p] = in ? a.lse[(int64_t)(h0 + i / kAtRows) * a.mq + row] : INFINITY;       // behind the end: p = 0
                delta_r[p] = in ? a.delta[(int64_t)(h0 + i / kAtRows) * a.mq + row] : 0.f;
            }
        };
#pragma unroll
        for (int h = 0; h < HG; ++h) slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] * kLog2e : 0.f;
        __syncthreads();                                       // the chunk of heads before has been read
        if (BIAS == kTable)
            for (int i = threadIdx.x; i < a.bias.buckets * HG; i += kAtBlock) table[i] = a.bias.table[(int64_t)(i / HG) * a.heads + h0 + i % HG] * kLog2e;
        if (first < last) fetch(first);
        for (int tile = first; tile < last; ++tile) {
            __syncthreads();
            ql.put_rows(qs);
            ql.put_cols(qt);
            gl.put_rows(gs);
            gl.put_cols(gt);
            if (BIAS != kNone && threadIdx.x < kAtRows) {
                cs[threadIdx.x] = (float)qc.y;
                cs[kAtRows + threadIdx.x] = (float)qc.z;
                cs[2 * kAtRows + threadIdx.x] = (float)qc.w;
            }
#pragma unroll
            for (int p = 0; p < (HG * kAtRows + kAtBlock - 1) / kAtBlock; ++p) {
                const int i = p * kAtBlock + threadIdx.x;
                if (i < HG * kAtRows) { ls[i] = lse_r[p] - AtType<T>::kLift; ds[i] = delta_r[p]; }
            }
            __syncthreads();
            if (tile + 1 < last) fetch(tile + 1);
            if (t.lo + wave * 16 >= t.hi) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float dist[8];
                int row_of[8];
                if (BIAS != kNone) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int at = 32 * j + 16 * b + 4 * g;
                        const f32x4 x = *reinterpret_cast<const f32x4*>(cs + at), y = *reinterpret_cast<const f32x4*>(cs + kAtRows + at),
                                    z = *reinterpret_cast<const f32x4*>(cs + 2 * kAtRows + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float dx = x[e] - kx, dy = y[e] - ky, dz = z[e] - kz, d2 = dx * dx + dy * dy + dz * dz;
                            if (BIAS == kSlope) dist[4 * b + e] = __builtin_amdgcn_sqrtf(d2);
                            if (BIAS == kTable) {
                                const AtCell c = cells[at_cell(d2)];
                                row_of[4 * b + e] = c.bucket + (d2 >= c.edge ? 1 : 0);
                            }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    const int slot = SLOTS == 1 ? 0 : h;
                    f32x4 s[2], dp[2];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
                        dp[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int c = 0; c < DC; ++c) {
                            const int at = h * Tile::kRows + (32 * j + 16 * b + col) * Tile::kRow + 32 * c + 8 * g;
                            at_mma(s[b], at_frag(qs + at), kf[slot][c]);
                            at_mma(dp[b], at_frag(gs + at), vf[slot][c]);
                        }
                        const f32x4 lse = *reinterpret_cast<const f32x4*>(ls + h * kAtRows + 32 * j + 16 * b + 4 * g),
                                    delta = *reinterpret_cast<const f32x4*>(ds + h * kAtRows + 32 * j + 16 * b + 4 * g);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = s[b][e] * scale2;
                            if (BIAS == kSlope) v += slope[h] * dist[4 * b + e];
                            if (BIAS == kTable) v += table[row_of[4 * b + e] * HG + h];
                            s[b][e] = __builtin_amdgcn_exp2f(v - lse[e]);
                            dp[b][e] = s[b][e] * (dp[b][e] - delta[e]);
                            if (kLifted) dp[b][e] *= ds_lift[slot];
                        }
                    }
                    Frag p, dsf;
                    at_pack(p, s[0], s[1]);
                    at_pack(dsf, dp[0], dp[1]);
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        const int at = h * Tile::kCols + (16 * b + col) * Tile::kCol + 32 * j + 4 * g;
                        at_mma(dv[slot][b], at_frag_rows(gt + at), p);
                        at_mma(dk[slot][b], at_frag_rows(qt + at), dsf);
                    }
                }
            }
        }
    }
    if (!have) return;
#pragma unroll
    for (int h = 0; h < SLOTS; ++h)
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            if (16 * b + 4 * g >= a.dim) continue;
            const int64_t at = ((int64_t)ki * kv_heads + kv0 + h) * a.dim + 16 * b + 4 * g;
            if (a.splits > 1) {
                const int64_t plane = (int64_t)a.mk * kv_heads * a.dim;
                at_store4(a.part_kv + (2 * split) * plane + at, dk[h][b] * dk_unlift[h]);
                at_store4(a.part_kv + (2 * split + 1) * plane + at, dv[h][b] * kUnlift);
            } else {
                at_store4((T*)a.dk + at, dk[h][b] * (a.scale * dk_unlift[h]));
                at_store4((T*)a.dv + at, dv[h][b] * kUnlift);
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
    typedef AtTile<T, DP> Tile;
    size_t lds = (size_t)SLOTS * (2 * Tile::kRows + Tile::kCols) * sizeof(T) + 3 * kAtRows * sizeof(float);
    if (BIAS == kTable) lds += (size_t)((a.bias.buckets * HG + 3) & ~3) * sizeof(float) + kCells * sizeof(AtCell);
    if (GRAD) lds += (size_t)4 * a.bias.buckets * HG * 64 * sizeof(float);
    const hipError_t e = hipFuncSetAttribute((const void*)at_bwd_q_kernel<T, DP, HG, SLOTS, BIAS, GRAD>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    at_bwd_q_kernel<T, DP, HG, SLOTS, BIAS, GRAD><<<(unsigned)((int64_t)a.tiles * (a.heads / HG)), kAtBlock, lds, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS, int BIAS>
static hipError_t at_bwd_kv_launch(const AtBwd& a, hipStream_t st) {
    typedef AtTile<T, DP> Tile;
    size_t lds = (size_t)HG * 2 * (Tile::kRows + Tile::kCols) * sizeof(T) + (3 + 2 * HG) * kAtRows * sizeof(float);
    if (BIAS == kTable) lds += (size_t)((a.bias.buckets * HG + 3) & ~3) * sizeof(float) + kCells * sizeof(AtCell);
    const hipError_t e = hipFuncSetAttribute((const void*)at_bwd_kv_kernel<T, DP, HG, SLOTS, BIAS>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    const int64_t wg = seg_tiles_bound(a.mk, kAtRows, a.seg_k, a.nseg) * (a.heads / a.share / SLOTS);
    at_bwd_kv_kernel<T, DP, HG, SLOTS, BIAS><<<dim3((unsigned)wg, (unsigned)a.splits), kAtBlock, lds, st>>>(a);
    if (a.splits > 1)
        at_join_kv_kernel<T><<<(unsigned)ceil_div((int64_t)a.mk * (a.heads / a.share) * a.dim / 4, 256), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS>
static hipError_t at_bwd_bias(const AtBwd& a, int mode, hipStream_t st) {
    hipError_t e = hipErrorInvalidValue;
    if (mode == kTable && a.part_t) e = at_bwd_q_launch<T, DP, 1, 1, kTable, true>(a, st);      // (the histogram leaves room for one head)
    else if (mode == kTable) e = at_bwd_q_launch<T, DP, HG, SLOTS, kTable, false>(a, st);
    else if (mode == kSlope) e = at_bwd_q_launch<T, DP, HG, SLOTS, kSlope, false>(a, st);
    else if constexpr (HG == 1) e = at_bwd_q_launch<T, DP, HG, SLOTS, kNone, false>(a, st);
    if (e != hipSuccess || a.dk == nullptr) return e;
    if (mode == kTable) return at_bwd_kv_launch<T, DP, HG, SLOTS, kTable>(a, st);
    if (mode == kSlope) return at_bwd_kv_launch<T, DP, HG, SLOTS, kSlope>(a, st);
    if constexpr (HG == 1) return at_bwd_kv_launch<T, DP, HG, SLOTS, kNone>(a, st);
    return hipErrorInvalidValue;
}

template <typename T>
static hipError_t at_bwd_dispatch(const AtBwd& a, int mode, hipStream_t st) {
    if (AtType<T>::kLift) {
        const int kv_heads = a.heads / a.share;
        at_bound_clear_kernel<<<(unsigned)ceil_div(2 * kv_heads, 256), 256, 0, st>>>(a.bound, 2 * kv_heads);
        at_bound_kernel<T><<<dim3((unsigned)ceil_div(a.mq, 256), (unsigned)a.heads), 256, 0, st>>>((const T*)a.go, a.go_row, a.go_head, a.mq, a.dim, a.share, a.bound);
        if (a.mk > 0)
            at_bound_kernel<T><<<dim3((unsigned)ceil_div(a.mk, 256), (unsigned)kv_heads), 256, 0, st>>>((const T*)a.v, a.v_row, a.v_head, a.mk, a.dim, 1,
                                                                                                    a.bound + kv_heads);
    }
    const int hg = at_heads_per_wave(a.dim, a.heads, a.share, mode);
    const bool one = a.share > 1;
    if (a.dim <= 32) {
        if (hg == 4) return one ? at_bwd_bias<T, 32, 4, 1>(a, mode, st) : at_bwd_bias<T, 32, 4, 4>(a, mode, st);
        return at_bwd_bias<T, 32, 1, 1>(a, mode, st);
    }
    if (a.dim <= 64) {
        if (hg == 2) return one ? at_bwd_bias<T, 64, 2, 1>(a, mode, st) : at_bwd_bias<T, 64, 2, 2>(a, mode, st);
        return at_bwd_bias<T, 64, 1, 1>(a, mode, st);
    }
    return at_bwd_bias<T, 128, 1, 1>(a, mode, st);
}

// shares of the queries for dk / dv, by the rule of the forward pass
static int at_bwd_splits(int64_t mq, int64_t mk, int nseg, int kv_heads, int slots) {
    const int64_t wg = (ceil_div(mk > 0 ? mk : 1, kAtRows) + (nseg > 1 ? nseg - 1 : 0)) * (kv_heads / slots);
    if (wg >= 512) return 1;
    const int64_t want = ceil_div(1024, wg), most = ceil_div(mq, nseg) / (4 * kAtRows);
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : (int)(n < 64 ? n : 64);
}

static int at_bwd_slots(int heads, int kv_heads, int dim, int mode) {
    const int share = heads / kv_heads;
    return share > 1 ? 1 : at_heads_per_wave(dim, heads, share, mode);
}

// workspace: delta and the bounds, the table's parts, the shares of dk / dv -- each on a 256-byte boundary
static int64_t at_bwd_layout(int64_t mq, int64_t mk, const void* seg, int64_t nseg, int heads, int kv_heads, int dim, int mode, int buckets, bool table_grad,
                             int64_t* off_t, int64_t* off_kv) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    *off_t = up((mq * heads + 2 * kv_heads) * (int64_t)sizeof(float));
    *off_kv = *off_t + (table_grad ? up(seg_tiles_bound(mq, kAtRows, seg, nseg) * heads * buckets * (int64_t)sizeof(float)) : 0);
    const int s = at_bwd_splits(mq, mk, (int)nseg, kv_heads, at_bwd_slots(heads, kv_heads, dim, mode));
    return *off_kv + (s > 1 ? up(2 * s * mk * kv_heads * dim * (int64_t)sizeof(float)) : 0);
}

}  // namespace lidiff

using namespace lidiff;

extern "C" int64_t lidiff_segment_attention_bwd_workspace_bytes(int64_t mq, int64_t mk, int64_t n_segments, int32_t heads, int32_t kv_heads, int32_t dim,
                                                                int32_t bias_mode, int32_t buckets, int32_t table_grad) {
    if (mq < 1 || mk < 0 || n_segments < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 128) return 0;
    int64_t t, kv;
    return at_bwd_layout(mq, mk, &t, n_segments, heads, kv_heads, dim, bias_mode, buckets, table_grad != 0, &t, &kv);      // (segments given: the larger bound)
}

extern "C" int lidiff_segment_attention_bwd(const void* q, const void* k, const void* v, const void* grad_out, const int64_t* strides,
                                            const int32_t* coords_q, const int32_t* coords_k, const int32_t* seg_q, const int32_t* seg_k,
                                            int64_t n_segments, int64_t mq, int64_t mk, int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype,
                                            float scale, int32_t bias_mode, const float* slopes, const float* table, const void* cells, int32_t buckets,
                                            const float* out_f32, const float* lse, void* dq, void* dk, void* dv, float* dtable, void* workspace,
                                            void* stream) {
    LIDIFF_CHECK_ARG(q && grad_out && strides && out_f32 && lse && dq && workspace && (mk == 0 || (k && v)) && (dk != nullptr) == (dv != nullptr), "null pointer");
    const char* bad = at_check(n_segments, mq, mk, heads, kv_heads, dim, dtype, bias_mode, buckets, strides, 8);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG((seg_q != nullptr) == (seg_k != nullptr) && (seg_q || n_segments == 1), "segments of queries and keys come together");
    LIDIFF_CHECK_ARG(bias_mode == kNone || (coords_q && (coords_k || mk == 0)), "a distance bias needs the coordinates");
    LIDIFF_CHECK_ARG(bias_mode != kSlope || slopes, "null pointer");
    LIDIFF_CHECK_ARG(bias_mode != kTable || (table && cells), "null pointer");
    LIDIFF_CHECK_ARG(dtable == nullptr || bias_mode == kTable, "a table gradient without a table");
    LIDIFF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)grad_out | (uintptr_t)out_f32 | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv |
                       (uintptr_t)coords_q | (uintptr_t)coords_k | (uintptr_t)workspace) & 15) == 0 &&
                     (((uintptr_t)seg_q | (uintptr_t)seg_k | (uintptr_t)cells) & 7) == 0, "misaligned pointer");
    AtBwd a;
    a.q = q; a.k = k; a.v = v; a.go = grad_out;
    a.q_row = strides[0]; a.q_head = strides[1]; a.k_row = strides[2]; a.k_head = strides[3]; a.v_row = strides[4]; a.v_head = strides[5];
    a.go_row = strides[6]; a.go_head = strides[7];
    a.cq = (const int4*)coords_q; a.ck = (const int4*)coords_k;
    a.seg_q = seg_q; a.seg_k = seg_k; a.nseg = (int)n_segments; a.mq = (int)mq; a.mk = (int)mk;
    a.heads = heads; a.share = heads / kv_heads; a.dim = dim;
    a.scale = scale;
    a.bias = AtBias{table, (const AtCell*)cells, slopes, buckets};
    a.out32 = out_f32; a.lse = lse;
    a.dq = dq; a.dk = mk > 0 ? dk : nullptr; a.dv = dv;
    int64_t off_t, off_kv;
    at_bwd_layout(mq, mk, seg_q, n_segments, heads, kv_heads, dim, bias_mode, buckets, dtable != nullptr, &off_t, &off_kv);
    a.delta = (float*)workspace;
    a.bound = (unsigned*)(a.delta + mq * heads);
    a.part_t = dtable ? (float*)((char*)workspace + off_t) : nullptr;
    a.part_kv = (float*)((char*)workspace + off_kv);
    a.tiles = (int)seg_tiles_bound(mq, kAtRows, seg_q, n_segments);
    a.splits = at_bwd_splits(mq, mk, a.nseg, kv_heads, at_bwd_slots(heads, kv_heads, dim, bias_mode));
    hipStream_t st = (hipStream_t)stream;
    LIDIFF_CHECK_HIP(dtype == 0 ? at_bwd_dispatch<float>(a, bias_mode, st) : dtype == 1 ? at_bwd_dispatch<__bf16>(a, bias_mode, st)
                                                                                      : at_bwd_dispatch<_Float16>(a, bias_mode, st));
    if (dtable) {
        at_table_kernel<<<(unsigned)(buckets * heads), kWave, 0, st>>>(a.part_t, a.tiles, heads, buckets, dtable);
        LIDIFF_CHECK_LAUNCH();
    }
    return 0;
}
