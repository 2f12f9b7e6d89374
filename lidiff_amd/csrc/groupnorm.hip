// Group normalisation with an activation over the rows of a feature matrix [M, C] (channels last), one statistic per (scan, group)
// for gfx950.  A scan is a row range of `segments` (segments.h); rows of no scan come out as zeros.
//   xh = (x - mean_sg) rstd_sg,   z = xh w_c + b_c,   y = act(z),     act: identity | max(z, 0) | z sigmoid(z)
//   backward, with dz = dy act'(z) and per (scan, channel) A_c = sum dz, B_c = sum dz xh over the scan's rows:
//   db_c = sum_s A_c,  dw_c = sum_s B_c,
//   dx = rstd (dz w_c - [sum_c' w_c' A_c' + xh sum_c' w_c' B_c'] / n)       (sums over the group's channels, n = rows x channels)
// HBM-bound, three launches a direction: partial sums of a slab of rows (one read of [M, C]), their sum in a fixed order, and the
// pass that writes.  The sums are held in double and taken of x less a value of the scan's (its first row's, one a group), so that the
// variance keeps its bits however far the mean is from zero; the mean is kept as two floats, whose first takes the leading bits off x exactly.
// Fixed orders: the same bits on every run.
#include "segments.h"

namespace lidiff {

constexpr int kGnBlock = 256;
constexpr int kGnSlabs = 1024;           // workgroups of a reduction over all scans together (4 per compute unit)
constexpr int kGnRowsPerThread = 16;     // rows a thread of the writing pass walks over, fewer where that would leave compute units idle

// rows of a workgroup of the writing pass (5 824 x 256, fp32: 9.2 us with 16 rows a thread, 8.5 with one)
static int gn_tile(int rows, int rpb) {
    const int n = rows / (rpb * kGnSlabs);
    return rpb * (n < 1 ? 1 : n < kGnRowsPerThread ? n : kGnRowsPerThread);
}

typedef __bf16 gn_bf16;
typedef _Float16 gn_f16;

template <typename T, int V>
struct alignas(sizeof(T) * V) GnVec { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void gn_load(const T* __restrict__ p, float (&f)[V]) {
    const GnVec<T, V> r = *reinterpret_cast<const GnVec<T, V>*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)r.v[e];
}

template <typename T, int V>
__device__ __forceinline__ void gn_store(T* __restrict__ p, const float (&f)[V]) {
    GnVec<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = (T)f[e];          // the output's own rounding, to nearest even
    *reinterpret_cast<GnVec<T, V>*>(p) = r;
}

__device__ __forceinline__ float gn_sigmoid(float z) {      // v_exp_f32 and v_rcp_f32: 1 ulp each
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
}

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
    return ACT == 0 ? z : ACT == 1 ? (z < 0.f ? 0.f : z) : z * gn_sigmoid(z);      // (a NaN stays one)
}

template <int ACT>
__device__ __forceinline__ float gn_act_slope(float z) {
    if (ACT == 0) return 1.f;
    if (ACT == 1) return z > 0.f ? 1.f : 0.f;
    const float s = gn_sigmoid(z);
    return s * (1.f + z * (1.f - s));
}

// where a thread stands: `cq` threads share a row, V channels each
template <int V>
struct GnLane {
    int cq, rl, q, rpb;
    bool on;
    __device__ GnLane(int c) : cq(c / V), rl(threadIdx.x / cq), q(threadIdx.x % cq), rpb(kGnBlock / cq), on(rl < rpb) {}
};

// slab `blk` of `nblk` of a segment's rows
__device__ __forceinline__ int2 gn_slab(int2 seg, int blk, int nblk) {
    const int64_t n = seg.y - seg.x;
    return make_int2(seg.x + (int)(n * blk / nblk), seg.x + (int)(n * (blk + 1) / nblk));
}

// sums of x - first and (x - first)^2 per (segment, group) over a slab: part[s][g][blk][2]; first: the value of the segment's first row in
// the group's first channel, which goes to stats[s][g].x
template <typename T, int V>
__global__ __launch_bounds__(kGnBlock) void gn_stats_kernel(const T* __restrict__ x, int rows, int c, int groups, const int32_t* __restrict__ seg,
                                                           int nblk, double* __restrict__ part, float4* __restrict__ stats) {
    extern __shared__ double gn_sm[];                                   // [rows per pass][c][2]
    const int s = blockIdx.x / nblk, blk = blockIdx.x % nblk, per = c / groups;
    const int2 all = seg_range(seg, s, rows), r = gn_slab(all, blk, nblk);
    const GnLane<V> at(c);
    double a[V] = {}, b[V] = {};
    if (at.on) {
        double from[V];
#pragma unroll
        for (int e = 0; e < V; ++e) from[e] = all.x < all.y ? (double)(float)x[(int64_t)all.x * c + (at.q * V + e) / per * per] : 0.0;
        for (int row = r.x + at.rl; row < r.y; row += at.rpb) {
            float f[V];
            gn_load<T, V>(x + (int64_t)row * c + at.q * V, f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double off = f[e] - from[e];
                a[e] += off;
                b[e] += off * off;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            gn_sm[(at.rl * c + at.q * V + e) * 2] = a[e];
            gn_sm[(at.rl * c + at.q * V + e) * 2 + 1] = b[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * c; i += kGnBlock) {               // over the row lanes, in order
        double t = 0;
        for (int l = 0; l < at.rpb; ++l) t += gn_sm[l * 2 * c + i];
        gn_sm[i] = t;                                                   // (row lane 0's own place: read by this thread only)
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * groups; i += kGnBlock) {          // over the group's channels, in order
        const int g = i >> 1;
        if (blk == 0 && i == 2 * g) stats[(int64_t)s * groups + g].x = all.x < all.y ? (float)x[(int64_t)all.x * c + g * per] : 0.f;      // (for the finish)
        double t = 0;
        for (int e = 0; e < per; ++e) t += gn_sm[(g * per + e) * 2 + (i & 1)];
        part[(((int64_t)s * groups + g) * nblk + blk) * 2 + (i & 1)] = t;
    }
}

// one wave per (segment, group): stats[s][g] = (mean's leading float, the rest of it, rstd, 0)
__global__ __launch_bounds__(kWave) void gn_finish_kernel(const double* __restrict__ part, int nblk, int rows, int c, int groups,
                                                           const int32_t* __restrict__ seg, float eps, float4* __restrict__ stats) {
    const int sg = blockIdx.x;
    double a = 0, b = 0;
    for (int i = threadIdx.x; i < nblk; i += kWave) {
        a += part[((int64_t)sg * nblk + i) * 2];
        b += part[((int64_t)sg * nblk + i) * 2 + 1];
    }
    for (int off = kWave / 2; off > 0; off >>= 1) { a += __shfl_down(a, off); b += __shfl_down(b, off); }
    if (threadIdx.x != 0) return;
    const int2 r = seg_range(seg, sg / groups, rows);
    const double n = (double)max(r.y - r.x, 1) * (c / groups), off = a / n, mean = stats[sg].x + off;
    double var = b / n - off * off;
    if (var < 0) var = 0;                                               // (a NaN passes)
    const float lead = (float)mean;
    stats[sg] = make_float4(lead, (float)(mean - lead), (float)(1.0 / sqrt(var + (double)eps)), 0.f);
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnBlock) void gn_apply_kernel(const T* __restrict__ x, int rows, int c, int groups, const int32_t* __restrict__ seg, int nseg,
                                                           int tile, const float4* __restrict__ stats, const float* __restrict__ w, const float* __restrict__ b,
                                                           T* __restrict__ y) {
    const GnLane<V> at(c);
    const SegTile t = find_seg_tile(seg, nseg, rows, tile, blockIdx.x);
    if (!at.on) return;
    float mean[V], scale[V], shift[V];
    const int per = c / groups;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int ch = at.q * V + e;
        const float4 st = t.seg >= 0 ? stats[(int64_t)t.seg * groups + ch / per] : make_float4(0.f, 0.f, 0.f, 0.f);
        mean[e] = st.x;
        scale[e] = st.z * (w ? w[ch] : 1.f);
        shift[e] = (b ? b[ch] : 0.f) - st.y * scale[e];
    }
    for (int row = t.lo + at.rl; row < t.hi; row += at.rpb) {
        float f[V] = {};
        if (t.seg >= 0) {
            gn_load<T, V>(x + (int64_t)row * c + at.q * V, f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = gn_act<ACT>((f[e] - mean[e]) * scale[e] + shift[e]);
        }
        gn_store<T, V>(y + (int64_t)row * c + at.q * V, f);
    }
}

// A_c and B_c over a slab: part[s][blk][2][c]
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnBlock) void gn_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy, int rows, int c, int groups,
                                                              const int32_t* __restrict__ seg, int nblk, const float4* __restrict__ stats,
                                                              const float* __restrict__ w, const float* __restrict__ b, double* __restrict__ part) {
    extern __shared__ double gn_sm[];
    const int s = blockIdx.x / nblk, blk = blockIdx.x % nblk;
    const int2 r = gn_slab(seg_range(seg, s, rows), blk, nblk);
    const GnLane<V> at(c);
    if (at.on) {
        double sa[V] = {}, sb[V] = {};
        float mean[V], less[V], rstd[V], wv[V], bv[V];                  // xh = (x - mean) rstd - less
        const int per = c / groups;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int ch = at.q * V + e;
            const float4 st = stats[(int64_t)s * groups + ch / per];
            mean[e] = st.x; rstd[e] = st.z; less[e] = st.y * st.z;
            wv[e] = w ? w[ch] : 1.f;
            bv[e] = b ? b[ch] : 0.f;
        }
        for (int row = r.x + at.rl; row < r.y; row += at.rpb) {
            float f[V], g[V];
            gn_load<T, V>(x + (int64_t)row * c + at.q * V, f);
            gn_load<T, V>(dy + (int64_t)row * c + at.q * V, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (f[e] - mean[e]) * rstd[e] - less[e];
                const float dz = g[e] * gn_act_slope<ACT>(xh * wv[e] + bv[e]);
                sa[e] += dz;
                sb[e] += (double)dz * xh;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            gn_sm[(at.rl * 2) * c + at.q * V + e] = sa[e];
            gn_sm[(at.rl * 2 + 1) * c + at.q * V + e] = sb[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * c; i += kGnBlock) {
        double t = 0;
        for (int l = 0; l < at.rpb; ++l) t += gn_sm[l * 2 * c + i];
        part[((int64_t)s * nblk + blk) * 2 * c + i] = t;
    }
}

// sums over the slabs: chan[s][2][c]; a workgroup takes 16 columns, 16 threads each walk over every 16th slab, joined in a fixed order
__global__ __launch_bounds__(256) void gn_bwd_finish_kernel(const double* __restrict__ part, int nblk, int c2, double* __restrict__ chan) {
    __shared__ double sm[16][17];
    const int cols = (c2 + 15) / 16, s = blockIdx.x / cols, col = (blockIdx.x % cols) * 16 + (threadIdx.x & 15), l = threadIdx.x >> 4;
    double t = 0;
    if (col < c2)
#pragma unroll 8
        for (int i = l; i < nblk; i += 16) t += part[((int64_t)s * nblk + i) * c2 + col];
    sm[l][threadIdx.x & 15] = t;
    __syncthreads();
    if (threadIdx.x < 16 && col < c2) {
        double u = 0;
        for (int i = 0; i < 16; ++i) u += sm[i][threadIdx.x];
        chan[(int64_t)s * c2 + col] = u;
    }
}

// the last workgroup of the grid adds the scans' A_c / B_c to db / dw; the others write dx
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnBlock) void gn_bwd_apply_kernel(const T* __restrict__ x, const T* __restrict__ dy, int rows, int c, int groups,
                                                               const int32_t* __restrict__ seg, int nseg, int tile, const float4* __restrict__ stats,
                                                               const double* __restrict__ chan, const float* __restrict__ w, const float* __restrict__ b,
                                                               T* __restrict__ dx, float* __restrict__ dw, float* __restrict__ db) {
    if (blockIdx.x == gridDim.x - 1) {
        for (int ch = threadIdx.x; ch < c; ch += kGnBlock) {
            double a = 0, bb = 0;
#pragma unroll 16
            for (int s = 0; s < nseg; ++s) { a += chan[(int64_t)s * 2 * c + ch]; bb += chan[((int64_t)s * 2 + 1) * c + ch]; }
            if (db) db[ch] = (float)a;
            if (dw) dw[ch] = (float)bb;
        }
        return;
    }
    __shared__ float sums[2 * 1024];                                    // per group: sum w A / n, sum w B / n
    const GnLane<V> at(c);
    const SegTile t = find_seg_tile(seg, nseg, rows, tile, blockIdx.x);
    if (t.lo >= t.hi) return;                                           // (the same for the whole workgroup)
    const int per = c / groups;
    if (t.seg >= 0) {
        const int2 r = seg_range(seg, t.seg, rows);
        const double inv_n = 1.0 / ((double)(r.y - r.x) * per);
        for (int i = threadIdx.x; i < 2 * groups; i += kGnBlock) {
            const int g = i >> 1;
            const double* src = chan + ((int64_t)t.seg * 2 + (i & 1)) * c + g * per;
            double u = 0;
            for (int e = 0; e < per; ++e) u += src[e] * (w ? (double)w[g * per + e] : 1.0);
            sums[i] = (float)(u * inv_n);
        }
    }
    __syncthreads();
    if (!at.on) return;
    float mean[V], less[V], rstd[V], wv[V], bv[V], ma[V], mb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int ch = at.q * V + e, g = ch / per;
        const float4 st = t.seg >= 0 ? stats[(int64_t)t.seg * groups + g] : make_float4(0.f, 0.f, 0.f, 0.f);
        mean[e] = st.x; rstd[e] = st.z; less[e] = st.y * st.z;
        wv[e] = w ? w[ch] : 1.f;
        bv[e] = b ? b[ch] : 0.f;
        ma[e] = t.seg >= 0 ? sums[2 * g] : 0.f;
        mb[e] = t.seg >= 0 ? sums[2 * g + 1] : 0.f;
    }
    for (int row = t.lo + at.rl; row < t.hi; row += at.rpb) {
        float f[V] = {};
        if (t.seg >= 0) {
            float g[V];
            gn_load<T, V>(x + (int64_t)row * c + at.q * V, f);
            gn_load<T, V>(dy + (int64_t)row * c + at.q * V, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (f[e] - mean[e]) * rstd[e] - less[e];
                const float dz = g[e] * gn_act_slope<ACT>(xh * wv[e] + bv[e]);
                f[e] = rstd[e] * (dz * wv[e] - ma[e] - xh * mb[e]);
            }
        }
        gn_store<T, V>(dx + (int64_t)row * c + at.q * V, f);
    }
}

static int gn_slabs(int64_t rows, int c, int v, int64_t nseg) {
    const int rpb = kGnBlock / (c / v);
    int64_t n = kGnSlabs / nseg;                                        // all scans together fill the card
    const int64_t most = ceil_div(ceil_div(rows, nseg), (int64_t)rpb * 8);      // >= 8 rows per thread of an average scan
    n = n < most ? n : most;
    return n < 1 ? 1 : (int)n;
}

template <typename T, int V, int ACT>
static void gn_fwd_launch(const void* x, int rows, int c, int groups, const int32_t* seg, int nseg, const float* w, const float* b, float eps, void* y,
                          float4* stats, double* ws, hipStream_t st) {
    const int nblk = gn_slabs(rows, c, V, nseg), rpb = kGnBlock / (c / V), tile = gn_tile(rows, rpb);
    gn_stats_kernel<T, V><<<(unsigned)(nseg * nblk), kGnBlock, (size_t)rpb * c * 2 * sizeof(double), st>>>((const T*)x, rows, c, groups, seg, nblk, ws, stats);
    gn_finish_kernel<<<(unsigned)(nseg * groups), kWave, 0, st>>>(ws, nblk, rows, c, groups, seg, eps, stats);
    gn_apply_kernel<T, V, ACT><<<(unsigned)seg_tiles_bound(rows, tile, seg, nseg), kGnBlock, 0, st>>>(
        (const T*)x, rows, c, groups, seg, nseg, tile, stats, w, b, (T*)y);
}

template <typename T, int V, int ACT>
static void gn_bwd_launch(const void* x, const void* dy, int rows, int c, int groups, const int32_t* seg, int nseg, const float4* stats, const float* w,
                          const float* b, void* dx, float* dw, float* db, double* ws, hipStream_t st) {
    const int nblk = gn_slabs(rows, c, V, nseg), rpb = kGnBlock / (c / V), tile = gn_tile(rows, rpb);
    double* chan = ws + (int64_t)nseg * nblk * 2 * c;
    gn_bwd_sums_kernel<T, V, ACT><<<(unsigned)(nseg * nblk), kGnBlock, (size_t)rpb * c * 2 * sizeof(double), st>>>((const T*)x, (const T*)dy, rows, c, groups, seg,
                                                                                                                nblk, stats, w, b, ws);
    gn_bwd_finish_kernel<<<(unsigned)(nseg * ((2 * c + 15) / 16)), 256, 0, st>>>(ws, nblk, 2 * c, chan);
    gn_bwd_apply_kernel<T, V, ACT><<<(unsigned)(seg_tiles_bound(rows, tile, seg, nseg) + 1), kGnBlock, 0, st>>>(
        (const T*)x, (const T*)dy, rows, c, groups, seg, nseg, tile, stats, chan, w, b, (T*)dx, dw, db);
}

// 16-byte accesses: 8 channels of a 16-bit type where C allows it, 4 otherwise
#define GN_DISPATCH(FN, ...)                                                                                          \
    do {                                                                                                              \
        if (dtype == 0) { GN_ACT(FN, float, 4, __VA_ARGS__); }                                                        \
        else if (dtype == 1 && c % 8 == 0) { GN_ACT(FN, gn_bf16, 8, __VA_ARGS__); }                                   \
        else if (dtype == 1) { GN_ACT(FN, gn_bf16, 4, __VA_ARGS__); }                                                 \
        else if (c % 8 == 0) { GN_ACT(FN, gn_f16, 8, __VA_ARGS__); }                                                  \
        else { GN_ACT(FN, gn_f16, 4, __VA_ARGS__); }                                                                  \
    } while (0)
#define GN_ACT(FN, T, V, ...)                                                                                         \
    do {                                                                                                              \
        if (act == 0) FN<T, V, 0>(__VA_ARGS__);                                                                       \
        else if (act == 1) FN<T, V, 1>(__VA_ARGS__);                                                                  \
        else FN<T, V, 2>(__VA_ARGS__);                                                                                \
    } while (0)

static const char* gn_check(int64_t rows, int c, int groups, int dtype, int64_t nseg, int act) {
    if (rows < 1 || rows > 0x7fffffff - 65536) return "need 1 <= rows < 2^31 - 65536";
    if (c < 4 || c > 1024 || c % 4) return "need a multiple of 4 channels in [4, 1024]";
    if (rows * c > (int64_t)1 << 33) return "need rows x channels <= 2^33";                  // (one launch's workgroups)
    if (groups < 1 || c % groups) return "the groups must divide the channels";
    if (dtype < 0 || dtype > 2) return "dtype: 0 fp32, 1 bf16, 2 fp16";
    if (nseg < 1 || nseg > 1 << 20) return "need 1 <= segments <= 2^20";
    if (nseg * groups > 1 << 25 || nseg * c > 1 << 26) return "need segments x groups <= 2^25, segments x channels <= 2^26";      // (likewise)
    if (act < 0 || act > 2) return "activation: 0 none, 1 relu, 2 silu";
    return nullptr;
}

}  // namespace lidiff

using namespace lidiff;

extern "C" int32_t lidiff_scanwise_version(void) { return 3; }

extern "C" int64_t lidiff_group_norm_workspace_bytes(int32_t c, int64_t n_segments) {
    const int64_t slabs = n_segments > kGnSlabs ? n_segments : kGnSlabs;               // of all scans together (gn_slabs)
    return (slabs + n_segments) * 2 * c * (int64_t)sizeof(double);
}

extern "C" int lidiff_group_norm(const void* x, int64_t rows, int32_t c, int32_t groups, int32_t dtype, const int32_t* segments, int64_t n_segments,
                                 const float* weight, const float* bias, float eps, int32_t act, void* y, float* stats, void* workspace, void* stream) {
    LIDIFF_CHECK_ARG(x && y && stats && workspace, "null pointer");
    const char* bad = gn_check(rows, c, groups, dtype, n_segments, act);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG(segments || n_segments == 1, "without segments all rows are one");
    LIDIFF_CHECK_ARG((((uintptr_t)x | (uintptr_t)y) & 15) == 0 && (((uintptr_t)segments | (uintptr_t)workspace) & 7) == 0 && ((uintptr_t)stats & 15) == 0, "misaligned pointer");
    const int nseg = (int)n_segments;
    GN_DISPATCH(gn_fwd_launch, x, (int)rows, c, groups, segments, nseg, weight, bias, eps, y, (float4*)stats, (double*)workspace, (hipStream_t)stream);
    LIDIFF_CHECK_LAUNCH();
    return 0;
}

extern "C" int lidiff_group_norm_bwd(const void* x, const void* dy, int64_t rows, int32_t c, int32_t groups, int32_t dtype, const int32_t* segments,
                                     int64_t n_segments, const float* weight, const float* bias, const float* stats, int32_t act, void* dx, float* dweight,
                                     float* dbias, void* workspace, void* stream) {
    LIDIFF_CHECK_ARG(x && dy && dx && stats && workspace, "null pointer");
    const char* bad = gn_check(rows, c, groups, dtype, n_segments, act);
    LIDIFF_CHECK_ARG(bad == nullptr, bad);
    LIDIFF_CHECK_ARG(segments || n_segments == 1, "without segments all rows are one");
    LIDIFF_CHECK_ARG((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)stats) & 15) == 0 && (((uintptr_t)segments | (uintptr_t)workspace) & 7) == 0,
                     "misaligned pointer");
    const int nseg = (int)n_segments;
    GN_DISPATCH(gn_bwd_launch, x, dy, (int)rows, c, groups, segments, nseg, (const float4*)stats, weight, bias, dx, dweight, dbias, (double*)workspace,
                (hipStream_t)stream);
    LIDIFF_CHECK_LAUNCH();
    return 0;
}

// -- the row ranges of a batch ------------------------------------------------------------------------------------------------------
namespace lidiff {
// rows grouped by ascending batch index: a row whose neighbour belongs to another batch writes its batch's boundary
__global__ void batch_segments_kernel(const int4* __restrict__ coords, int64_t rows, const int32_t* __restrict__ d_rows, int nb, int replicas,
                                      int2* __restrict__ seg, int32_t* __restrict__ status) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t n = d_rows ? min(rows, (int64_t)max(*d_rows, 0)) : rows;
    if (i >= n) return;
    const int b = coords[i].x, before = i > 0 ? coords[i - 1].x : -1, behind = i + 1 < n ? coords[i + 1].x : nb;
    if (b < 0 || b >= nb || b < before) { atomicOr(status, LIDIFF_STATUS_BATCH_ORDER); return; }
    for (int r = 0; r < replicas; ++r) {                                // a replica's rows start at r * rows (the bound), gaps between
        int2* out = seg + (int64_t)r * nb + b;
        if (b != before) out->x = (int)(r * rows + i);
        if (b != behind) out->y = (int)(r * rows + i + 1);
    }
}
}  // namespace lidiff

extern "C" int lidiff_batch_segments(const int32_t* coords, int64_t rows, const int32_t* d_rows, int32_t n_batches, int32_t replicas, int32_t* segments,
                                     int32_t* status, void* stream) {
    LIDIFF_CHECK_ARG(segments && status && (coords || rows == 0), "null pointer");
    LIDIFF_CHECK_ARG(rows >= 0 && n_batches >= 1 && replicas >= 1 && rows * replicas < (int64_t)1 << 31, "need rows * replicas < 2^31, batches and replicas >= 1");
    LIDIFF_CHECK_ARG(((uintptr_t)coords & 15) == 0 && ((uintptr_t)segments & 7) == 0, "misaligned pointer");
    if (rows == 0) return 0;
    batch_segments_kernel<<<(unsigned)ceil_div(rows, 256), 256, 0, (hipStream_t)stream>>>((const int4*)coords, rows, d_rows, n_batches, replicas, (int2*)segments,
                                                                                        status);
    LIDIFF_CHECK_LAUNCH();
    return 0;
}
