// Attention between the rows of the same scan, forward: out_i = sum_j softmax_j(q_i . k_j scale + bias_h(|c_i - c_j|)) v_j over the keys j of
// i's scan (segments.h), in one pass over the keys with a running maximum and sum per query and head.  A query whose scan has no keys,
// and a row of no scan, gives zeros.
// Scores are kept in units of log 2 (scale, slopes and table times log2 e), so a probability is one v_exp_f32.
#include "attention.h"

namespace lidiff {

struct AtFwd {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;      // strides in elements
    const int4 *cq, *ck;                                      // (batch, x, y, z) of every row, for the biases
    const int32_t *seg_q, *seg_k;
    int nseg, mq, mk, heads, share, dim;                      // share: query heads per key head
    float scale;                                              // already times log2 e
    AtBias bias;
    int splits;                                               // the keys of a scan are shared out over `splits` workgroups
    void* out;                                                // [mq][heads][dim]
    float* out32;                                             // the same unrounded (for the backward pass), or null
    int exact;                                                // probabilities in pieces: out32 is wanted to fp32 precision
    float* lse;                                               // [heads][mq]: log2 of the sum of exponentials, +inf for a row without keys; or null
    float *part_o, *part_ml;                                  // splits > 1: [splits][mq][heads][dim], [splits][2][heads][mq]
};

// one workgroup: 64 queries of one scan (16 a wave) x HG heads x one share of the keys.
// EXACT (16-bit operands, when the table's gradient is wanted): probabilities enter the product with the values in pieces, rounding and
// rest.  d table sums ds over millions of pairs whose rows cancel to zero through delta = do . out, so an output from probabilities of 8 or
// 11 bits costs it more than fp32 sums do.
template <typename T, int DP, int HG, int SLOTS, int BIAS, bool EXACT>
__global__ __launch_bounds__(kAtBlock) void at_fwd_kernel(const AtFwd a) {
    typedef AtTile<T, DP> Tile;
    typedef typename AtType<T>::Frag Frag;
    constexpr int DC = DP / 32, DB = DP / 16;
    constexpr float kLift = AtType<T>::kLift, kUnlift = AtType<T>::kLift ? 1.f / (1 << AtType<T>::kLift) : 1.f;
    extern __shared__ __align__(16) unsigned char at_sm[];
    T* ks = reinterpret_cast<T*>(at_sm);                                          // keys, row by row
    T* vs = ks + SLOTS * Tile::kRows;                                             // values, transposed
    float* cs = reinterpret_cast<float*>(vs + SLOTS * Tile::kCols);               // x, y, z of the tile's keys
    float* table = cs + 3 * kAtRows;                                              // [buckets][HG]
    AtCell* cells = reinterpret_cast<AtCell*>(table + (BIAS == kTable ? ((a.bias.buckets * HG + 3) & ~3) : 0));

    const int lane = lane_id(), wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const int groups = a.heads / HG, h0 = (blockIdx.x % groups) * HG, kv0 = h0 / a.share, split = blockIdx.y;
    const SegTile t = find_seg_tile(a.seg_q, a.nseg, a.mq, kAtRows, blockIdx.x / groups);
    if (t.lo >= t.hi) return;
    const int qi = t.lo + wave * 16 + col;
    const bool have = qi < t.hi;
    const int2 kr = t.seg >= 0 ? seg_range(a.seg_k, t.seg, a.mk) : make_int2(0, 0);
    const int tiles = (kr.y - kr.x + kAtRows - 1) / kAtRows;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);

    Frag qf[HG][DC];
#pragma unroll
    for (int h = 0; h < HG; ++h)
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = 32 * c + 8 * g;
            qf[h][c] = have && d < a.dim ? at_frag((const T*)a.q + (int64_t)qi * a.q_row + (int64_t)(h0 + h) * a.q_head + d) : at_zero<T>();
        }
    float qx = 0.f, qy = 0.f, qz = 0.f, slope[HG];
    if (BIAS != kNone && have) {
        const int4 c = a.cq[qi];
        qx = (float)c.y; qy = (float)c.z; qz = (float)c.w;
    }
#pragma unroll
    for (int h = 0; h < HG; ++h) slope[h] = BIAS == kSlope ? -a.bias.slopes[h0 + h] * kLog2e : 0.f;
    if (BIAS == kTable) {
        for (int i = threadIdx.x; i < a.bias.buckets * HG; i += kAtBlock) table[i] = a.bias.table[(int64_t)(i / HG) * a.heads + h0 + i % HG] * kLog2e;
        for (int i = threadIdx.x; i < kCells; i += kAtBlock) cells[i] = a.bias.cells[i];
    }

    f32x4 o[HG][DB] = {};
    float m[HG], l[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) { m[h] = -INFINITY; l[h] = 0.f; }

    AtLoad<T, DP, SLOTS> kl, vl;
    int4 kc = make_int4(0, 0, 0, 0);
    auto fetch = [&](int tile) {
        const int lo = kr.x + tile * kAtRows;
        kl.fetch((const T*)a.k, a.k_row, a.k_head, kv0, a.dim, lo, kr.y);
        vl.fetch((const T*)a.v, a.v_row, a.v_head, kv0, a.dim, lo, kr.y);
        if (BIAS != kNone && threadIdx.x < kAtRows && lo + (int)threadIdx.x < kr.y) kc = a.ck[lo + threadIdx.x];
    };
    if (first < last) fetch(first);
    for (int tile = first; tile < last; ++tile) {
        __syncthreads();                                       // the tile before has been read
        kl.put_rows(ks);
        vl.put_cols(vs);
        if (BIAS != kNone && threadIdx.x < kAtRows) {
            cs[threadIdx.x] = (float)kc.y;
            cs[kAtRows + threadIdx.x] = (float)kc.z;
            cs[2 * kAtRows + threadIdx.x] = (float)kc.w;
        }
        __syncthreads();
        if (tile + 1 < last) fetch(tile + 1);                  // in flight under the products
        if (t.lo + wave * 16 >= t.hi) continue;                // a wave without queries only loads
        const int left = kr.y - (kr.x + tile * kAtRows);       // keys of this tile, 64 except at the end

        // what the heads share: distance, or the offset of the bucket's row in the table
        float dist[16];
        int row_of[16];
        if (BIAS != kNone) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(cs + 16 * b + 4 * g), y = *reinterpret_cast<const f32x4*>(cs + kAtRows + 16 * b + 4 * g),
                            z = *reinterpret_cast<const f32x4*>(cs + 2 * kAtRows + 16 * b + 4 * g);
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
            f32x4 s[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < DC; ++c) at_mma(s[b], at_frag(ks + slot * Tile::kRows + (16 * b + col) * Tile::kRow + 32 * c + 8 * g), qf[h][c]);
            }
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = s[b][e] * a.scale;
                    if (BIAS == kSlope) v += slope[h] * dist[4 * b + e];
                    if (BIAS == kTable) v += table[row_of[4 * b + e] * HG + h];
                    if (left < kAtRows && 16 * b + 4 * g + e >= left) v = -INFINITY;
                    s[b][e] = v;
                    top = fmaxf(top, v);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float now = fmaxf(m[h], top), safe = now == -INFINITY ? 0.f : now, base = safe - kLift;
            const float fade = __builtin_amdgcn_exp2f(m[h] - safe);
            m[h] = now;
            l[h] *= fade;
#pragma unroll
            for (int b = 0; b < DB; ++b) o[h][b] *= fade;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[b][e] = __builtin_amdgcn_exp2f(s[b][e] - base);
                    l[h] += s[b][e];
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                constexpr int PIECES = EXACT ? AtType<T>::kPieces : 1;
                Frag p[PIECES];
                at_pack(p[0], s[2 * j], s[2 * j + 1]);
                if constexpr (PIECES > 1) {
#pragma unroll
                    for (int i = 1; i < PIECES; ++i) at_pack_rest(p[i], p[i - 1], s[2 * j], s[2 * j + 1]);
                }
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    const Frag vf = at_frag_rows(vs + slot * Tile::kCols + (16 * b + col) * Tile::kCol + 32 * j + 4 * g);
#pragma unroll
                    for (int i = 0; i < PIECES; ++i) at_mma(o[h][b], vf, p[i]);
                }
            }
        }
    }
    if (!have) return;
#pragma unroll
    for (int h = 0; h < HG; ++h) {
        float sum = l[h] + __shfl_xor(l[h], 16);               // (the four lanes of a query leave together: `have` is the same for them)
        sum += __shfl_xor(sum, 32);
        const int head = h0 + h;
        if (a.splits > 1) {
            if (g == 0) {
                a.part_ml[((int64_t)(2 * split) * a.heads + head) * a.mq + qi] = m[h];
                a.part_ml[((int64_t)(2 * split + 1) * a.heads + head) * a.mq + qi] = sum * kUnlift;
            }
#pragma unroll
            for (int b = 0; b < DB; ++b)
                if (16 * b + 4 * g < a.dim) at_store4(a.part_o + (((int64_t)split * a.mq + qi) * a.heads + head) * a.dim + 16 * b + 4 * g, o[h][b] * kUnlift);
            continue;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (a.lse && g == 0) a.lse[(int64_t)head * a.mq + qi] = sum == 0.f ? INFINITY : m[h] - kLift + log2f(sum);
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            if (16 * b + 4 * g >= a.dim) continue;
            const f32x4 r = o[h][b] * inv;
            const int64_t at = ((int64_t)qi * a.heads + head) * a.dim + 16 * b + 4 * g;
            at_store4((T*)a.out + at, r);
            if (a.out32) at_store4(a.out32 + at, r);
        }
    }
}

// joins the shares of the keys: a thread takes four elements of one (query, head)
template <typename T>
__global__ void at_join_kernel(const AtFwd a) {
    const int quads = a.dim / 4;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, total = (int64_t)a.mq * a.heads * quads;
    if (i >= total) return;
    const int d = (int)(i % quads) * 4, head = (int)(i / quads % a.heads), qi = (int)(i / quads / a.heads);
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[((int64_t)(2 * s) * a.heads + head) * a.mq + qi]);
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float w = __builtin_amdgcn_exp2f(a.part_ml[((int64_t)(2 * s) * a.heads + head) * a.mq + qi] - base);
        sum += w * a.part_ml[((int64_t)(2 * s + 1) * a.heads + head) * a.mq + qi];
        const f32x4 p = *reinterpret_cast<const f32x4*>(a.part_o + (((int64_t)s * a.mq + qi) * a.heads + head) * a.dim + d);
        o += w * p;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const f32x4 r = o * inv;
    const int64_t at = ((int64_t)qi * a.heads + head) * a.dim + d;
    at_store4((T*)a.out + at, r);
    if (a.out32) at_store4(a.out32 + at, r);
    if (a.lse && d == 0) a.lse[(int64_t)head * a.mq + qi] = sum == 0.f ? INFINITY : m + log2f(sum);
}

template <typename T, int DP, int HG, int SLOTS, int BIAS, bool EXACT = false>
static hipError_t at_fwd_launch(const AtFwd& a, hipStream_t st) {
    typedef AtTile<T, DP> Tile;
    const int64_t wg = seg_tiles_bound(a.mq, kAtRows, a.seg_q, a.nseg) * (a.heads / HG);
    size_t lds = (size_t)SLOTS * (Tile::kRows + Tile::kCols) * sizeof(T) + 3 * kAtRows * sizeof(float);
    if (BIAS == kTable) lds += (size_t)((a.bias.buckets * HG + 3) & ~3) * sizeof(float) + kCells * sizeof(AtCell);
    const hipError_t e = hipFuncSetAttribute((const void*)at_fwd_kernel<T, DP, HG, SLOTS, BIAS, EXACT>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    at_fwd_kernel<T, DP, HG, SLOTS, BIAS, EXACT><<<dim3((unsigned)wg, (unsigned)a.splits), kAtBlock, lds, st>>>(a);
    if (a.splits > 1) at_join_kernel<T><<<(unsigned)ceil_div((int64_t)a.mq * a.heads * (a.dim / 4), 256), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int HG, int SLOTS>
static hipError_t at_fwd_bias(const AtFwd& a, int mode, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (mode == kTable && a.exact) return at_fwd_launch<T, DP, HG, SLOTS, kTable, true>(a, st);
    if (mode == kTable) return at_fwd_launch<T, DP, HG, SLOTS, kTable>(a, st);
    if (mode == kSlope) return at_fwd_launch<T, DP, HG, SLOTS, kSlope>(a, st);
    if constexpr (HG == 1) return at_fwd_launch<T, DP, HG, SLOTS, kNone>(a, st);
    return hipErrorInvalidValue;
}

template <typename T>
static hipError_t at_fwd_dispatch(const AtFwd& a, int mode, hipStream_t st) {
    const int hg = at_heads_per_wave(a.dim, a.heads, a.share, mode);
    const bool one = a.share > 1;
    if (a.dim <= 32) {
        if (hg == 4) return one ? at_fwd_bias<T, 32, 4, 1>(a, mode, st) : at_fwd_bias<T, 32, 4, 4>(a, mode, st);
        return at_fwd_bias<T, 32, 1, 1>(a, mode, st);
    }
    if (a.dim <= 64) {
        if (hg == 2) return one ? at_fwd_bias<T, 64, 2, 1>(a, mode, st) : at_fwd_bias<T, 64, 2, 2>(a, mode, st);
        return at_fwd_bias<T, 64, 1, 1>(a, mode, st);
    }
    return at_fwd_bias<T, 128, 1, 1>(a, mode, st);
}

// how many workgroups share a scan's keys: one while there are workgroups enough for the card, else so many that there are, each with
// at least four tiles of an average scan's keys
static int at_fwd_splits(int64_t mq, int64_t mk, int nseg, int heads, int hg) {
    const int64_t wg = (ceil_div(mq, kAtRows) + (nseg > 1 ? nseg - 1 : 0)) * (heads / hg);
    if (wg >= 512) return 1;
    const int64_t want = ceil_div(1024, wg), most = ceil_div(mk, nseg) / (4 * kAtRows);
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : (int)(n < 64 ? n : 64);
}

}  // namespace lidiff

using namespace lidiff;

extern "C" int64_t lidiff_segment_attention_workspace_bytes(int64_t mq, int64_t mk, int64_t n_segments, int32_t heads, int32_t kv_heads, int32_t dim,
                                                            int32_t bias_mode) {
    if (mq < 1 || n_segments < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 128) return 0;
    const int s = at_fwd_splits(mq, mk, (int)n_segments, heads, at_heads_per_wave(dim, heads, heads / kv_heads, bias_mode));
    return s == 1 ? 0 : (int64_t)s * mq * heads * (dim + 2) * (int64_t)sizeof(float);
}

extern "C" int lidiff_segment_attention(const void* q, const void* k, const void* v, const int64_t* strides, const int32_t* coords_q, const int32_t* coords_k,
                                        const int32_t* seg_q, const int32_t* seg_k, int64_t n_segments, int64_t mq, int64_t mk, int32_t heads,
                                        int32_t kv_heads, int32_t dim, int32_t dtype, float scale, int32_t bias_mode, const float* slopes,
                                        const float* table, const void* cells, int32_t buckets, void* out, float* out_f32, int32_t exact, float* lse,
                                        void* workspace,
                                        void* stream) {
    LIDIFF_CHECK_ARG(q && out && strides && (mk == 0 || (k && v)), "null pointer");
    const char* bad = at_check(n_segments, mq, mk, heads, kv_heads, dim, dtype, bias_mode, buckets, strides, 6);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG((seg_q != nullptr) == (seg_k != nullptr) && (seg_q || n_segments == 1), "segments of queries and keys come together");
    LIDIFF_CHECK_ARG(bias_mode == kNone || (coords_q && (coords_k || mk == 0)), "a distance bias needs the coordinates");
    LIDIFF_CHECK_ARG(bias_mode != kSlope || slopes, "null pointer");
    LIDIFF_CHECK_ARG(bias_mode != kTable || (table && cells), "null pointer");
    LIDIFF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)out_f32 | (uintptr_t)coords_q | (uintptr_t)coords_k |
                       (uintptr_t)workspace) & 15) == 0 && (((uintptr_t)seg_q | (uintptr_t)seg_k | (uintptr_t)cells) & 7) == 0, "misaligned pointer");
    AtFwd a;
    a.q = q; a.k = k; a.v = v;
    a.q_row = strides[0]; a.q_head = strides[1]; a.k_row = strides[2]; a.k_head = strides[3]; a.v_row = strides[4]; a.v_head = strides[5];
    a.cq = (const int4*)coords_q; a.ck = (const int4*)coords_k;
    a.seg_q = seg_q; a.seg_k = seg_k; a.nseg = (int)n_segments; a.mq = (int)mq; a.mk = (int)mk;
    a.heads = heads; a.share = heads / kv_heads; a.dim = dim;
    a.scale = scale * kLog2e;
    a.bias = AtBias{table, (const AtCell*)cells, slopes, buckets};
    a.splits = at_fwd_splits(mq, mk, a.nseg, heads, at_heads_per_wave(dim, heads, a.share, bias_mode));
    a.out = out; a.out32 = out_f32; a.exact = exact; a.lse = lse;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o ? a.part_o + (int64_t)a.splits * mq * heads * dim : nullptr;
    LIDIFF_CHECK_ARG(a.splits == 1 || workspace, "workspace missing (lidiff_segment_attention_workspace_bytes)");
    hipStream_t st = (hipStream_t)stream;
    LIDIFF_CHECK_HIP(dtype == 0 ? at_fwd_dispatch<float>(a, bias_mode, st) : dtype == 1 ? at_fwd_dispatch<__bf16>(a, bias_mode, st)
                                                                                      : at_fwd_dispatch<_Float16>(a, bias_mode, st));
    return 0;
}
