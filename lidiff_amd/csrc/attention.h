// Pieces shared by the attention kernels (attention_fwd.hip, attention_bwd.hip): operands, matrix products, row tiles in LDS, distance
// biases.
//
// One wave owns 16 or 32 "columns" (queries, or keys in the dk / dv kernel) of HG heads and walks over tiles of "rows" of the other side.
// A product S = X Y^T in 16 x 16 blocks of v_mfma_f32_16x16x32 leaves in lane l the column l & 15 and the rows 4 (l >> 4) .. + 3 of a
// block: a column's statistics live in its own lanes, and the block IS (after rounding to the operands' type) half of the B operand of the
// next product over the rows -- no value crosses a lane.  A contraction may take its terms in any order as long as both operands agree, so
// rows 32 j + 16 (e / 4) + 4 g + e % 4 are the terms 8 g + e of lane group g = l >> 4 of product j; the A operand with exactly these rows
// is read from the same row-major tile by the transposing LDS read, so a tile is held once.
#pragma once
#include "segments.h"

namespace lidiff {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* at_lds_t;
typedef uint32_t at_words __attribute__((ext_vector_type(4)));

constexpr int kAtBlock = 256;      // 4 waves; two a SIMD (at_waves): with at most 256 registers the matrix results stay in vector registers
constexpr float kLog2e = 1.44269504088896340736f;

// -- operands -----------------------------------------------------------------------------------------------------------------------
// fp32 tensors enter the matrix pipe as three bf16 pieces x = x0 + x1 + x2 (exact: 8 + 8 + 8 bits); of the nine products the six that
// reach 2^-24 |x y| are formed: fp32 accuracy in 6 / 16 of the time of the fp32 matrix instruction.
// kLift: fp16 ends at 2^-24, where a probability of a long scan may well lie.  Probabilities are multiplied by a power of two before they
// are rounded to an fp16 operand and the sums divided by it -- exact, and an addend of an exponent that is formed anyway.
struct AtPieces { bf16x8 p[3]; };
template <typename T> struct AtType;
// waves a SIMD the kernels are compiled for (the widest fp32 rows need more than 256 registers)
constexpr int at_waves(int bytes, int width) { return bytes == 4 && width == 128 ? 1 : 2; }
template <> struct AtType<__bf16> { typedef bf16x8 Frag; typedef bf16x4 Quad; typedef __bf16 Elem; static constexpr int kPlanes = 1, kLift = 0, kPieces = 3; };
template <> struct AtType<_Float16> { typedef f16x8 Frag; typedef f16x4 Quad; typedef _Float16 Elem; static constexpr int kPlanes = 1, kLift = 15, kPieces = 2; };
template <> struct AtType<float> { typedef AtPieces Frag; typedef f32x4 Quad; typedef __bf16 Elem; static constexpr int kPlanes = 3, kLift = 0, kPieces = 1; };

// acc += A B over 32 terms: lane group g holds the terms 8 g .. 8 g + 7 of row (A) / column (B) lane & 15
__device__ __forceinline__ void at_mma(f32x4& acc, const bf16x8& a, const bf16x8& b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void at_mma(f32x4& acc, const f16x8& a, const f16x8& b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void at_mma(f32x4& acc, const AtPieces& a, const AtPieces& b) {
    at_mma(acc, a.p[0], b.p[2]); at_mma(acc, a.p[1], b.p[1]); at_mma(acc, a.p[2], b.p[0]);
    at_mma(acc, a.p[0], b.p[1]); at_mma(acc, a.p[1], b.p[0]); at_mma(acc, a.p[0], b.p[0]);
}

// the same with the parts joined by ordinary additions: the matrix pipe rounds a chain of sums to one side, which a sum over 10^8 values
// that cancel does not forgive
template <typename F>
__device__ __forceinline__ void at_mma_apart(f32x4& acc, const F& a, const F& b) {
    f32x4 part = {0.f, 0.f, 0.f, 0.f};
    at_mma(part, a, b);
    acc += part;
}
__device__ __forceinline__ void at_mma_apart(f32x4& acc, const AtPieces& a, const AtPieces& b) {
    f32x4 low = {0.f, 0.f, 0.f, 0.f}, part = low;
    at_mma(low, a.p[0], b.p[2]); at_mma(low, a.p[1], b.p[1]); at_mma(low, a.p[2], b.p[0]);
    at_mma(low, a.p[0], b.p[1]); at_mma(low, a.p[1], b.p[0]);
    at_mma(part, a.p[0], b.p[0]);
    acc += low;
    acc += part;
}

// sums over the rows of a scan: fp32 operands have every 32 rows summed by themselves, so that the cuts do not add up along the chain; with
// 16-bit operands they are far below the operands' rounding
template <typename F>
__device__ __forceinline__ void at_mma_rows(f32x4& acc, const F& a, const F& b) { at_mma(acc, a, b); }
__device__ __forceinline__ void at_mma_rows(f32x4& acc, const AtPieces& a, const AtPieces& b) {
    f32x4 part = {0.f, 0.f, 0.f, 0.f};
    at_mma(part, a, b);
    acc += part;
}

// the operand with its signs turned where `mask` is 0x80008000
__device__ __forceinline__ void at_turn(bf16x8& f, uint32_t mask) { f = __builtin_bit_cast(bf16x8, __builtin_bit_cast(at_words, f) ^ mask); }
__device__ __forceinline__ void at_turn(f16x8& f, uint32_t mask) { f = __builtin_bit_cast(f16x8, __builtin_bit_cast(at_words, f) ^ mask); }
__device__ __forceinline__ void at_turn(AtPieces& f, uint32_t mask) {
#pragma unroll
    for (int i = 0; i < 3; ++i) at_turn(f.p[i], mask);
}

// x into its pieces; a value that is not finite goes into the first alone (so that it stays what it is), and one that rounds beyond
// bf16's largest is cut to it first
__device__ __forceinline__ void at_split(float x, __bf16& p0, __bf16& p1, __bf16& p2) {
    const float big = 3.38953139e38f;
    const bool finite = fabsf(x) < INFINITY;
    p0 = (__bf16)(finite ? fminf(fmaxf(x, -big), big) : x);
    const float r = finite ? x - (float)p0 : 0.f;
    p1 = (__bf16)r;
    p2 = (__bf16)(r - (float)p1);
}

// eight consecutive elements of a row as an operand
__device__ __forceinline__ bf16x8 at_load8(const __bf16* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ f16x8 at_load8(const _Float16* p) { return *reinterpret_cast<const f16x8*>(p); }
__device__ __forceinline__ AtPieces at_load8(const float* p) {
    AtPieces f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        __bf16 a, b, c;
        at_split(p[e], a, b, c);
        f.p[0][e] = a; f.p[1][e] = b; f.p[2][e] = c;
    }
    return f;
}

// two accumulator blocks (rows 32 j .. + 15 and + 16 .. + 31) as the B operand of the next product.  For 16-bit operands this rounds the
// probabilities (or their gradients) once, to the type the other operand has: the matrix instruction takes one type.
__device__ __forceinline__ f32x8 at_join(const f32x4& a, const f32x4& b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ void at_pack(bf16x8& f, const f32x8& v) { f = __builtin_convertvector(v, bf16x8); }
__device__ __forceinline__ void at_pack(f16x8& f, const f32x8& v) { f = __builtin_convertvector(v, f16x8); }
__device__ __forceinline__ void at_pack(AtPieces& f, const f32x8& v) {
    at_pack(f.p[0], v);
    const f32x8 r = v - __builtin_convertvector(f.p[0], f32x8);
    at_pack(f.p[1], r);
    at_pack(f.p[2], r - __builtin_convertvector(f.p[1], f32x8));
}
// what the rounding of at_pack left (v: the values on entry, what is still left on return), as a further operand
template <typename F>
__device__ __forceinline__ void at_pack_rest(F& rest, const F& piece, f32x8& v) {
    v -= __builtin_convertvector(piece, f32x8);
    at_pack(rest, v);
}

// a value that only the branch it stands in knows: keeps a rarely taken branch a branch (the compiler would turn it into selections that
// every pass pays for)
__device__ __forceinline__ int at_here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ void at_here(f32x4& v) { asm volatile("" : "+v"(v)); }

// A probability is exp2(s scale2 - base) with one rounding (fma).  Where the base is so large (|base| > 2^20, where fp32 steps by 1/8) that
// the rounding of the base alone is a factor, the product is rounded first, so that the scores the base was formed from give 1.
constexpr float kHuge = 1048576.f;
__device__ __forceinline__ bool at_huge(float base) { return __any(fabsf(base) > kHuge && fabsf(base) < INFINITY); }
__device__ __forceinline__ float at_exponent(float s, float scale2, float base) {
    float product = __fmul_rn(s, scale2);
    asm volatile("" : "+v"(product));                          // (no fma of it and the subtraction)
    return fabsf(base) > kHuge ? product - base : __fmaf_rn(s, scale2, -base);
}

// The log2 of a sum of exponentials is base + log2(sum), kept as two numbers whose sum is exact: one fp32 number steps by 2^-23 |base|, and a
// probability rebuilt from it is off by that factor (13 equal scores of 2^14: 5e-4; of 2^22: 15 %).  The backward pass's exponent is
// s scale2 - lse.  Up to |lse| = 2^6 the first number alone does (2^-19 of rounding: 1.3e-6 of the row's probabilities, alike for all of
// them); beyond, in a wave that has such a row, the product less the first number is small, and the second one is subtracted from that.
constexpr float kFar = 64.f;
__device__ __forceinline__ bool at_far(float lse) { return __any(fabsf(lse) > kFar && fabsf(lse) < INFINITY); }
__device__ __forceinline__ float at_two_sum(float a, float b, float& rest) {
    const float sum = a + b, part = sum - a;
    rest = fabsf(sum) < INFINITY ? (a - (sum - part)) + (b - part) : 0.f;
    return sum;
}

// four consecutive outputs
template <typename T>
__device__ __forceinline__ void at_store4(T* p, const f32x4& v) {
    typedef typename AtType<T>::Quad Quad;
    *reinterpret_cast<Quad*>(p) = __builtin_convertvector(v, Quad);
}

// -- row tiles ------------------------------------------------------------------------------------------------------------------------
// a tensor as the kernels stream it: rows of DP 16-bit elements; strides in bytes; fp32 tensors come as three planes
struct AtRows {
    const char* p;
    int64_t row, head, plane;
};

// ROWS rows x SLOTS heads x planes in LDS without padding, 16-byte pieces.  Piece c of a row stands at c ^ swz(row): sixteen rows read at
// one piece (b128, the A operand as it is) and four rows read at a pair of pieces (the transposing read) each touch every bank alike.
template <typename T, int DP, int SLOTS, int ROWS>
struct AtTile {
    typedef typename AtType<T>::Frag Frag;
    static constexpr int P = AtType<T>::kPlanes;
    static constexpr int CH = DP / 8;                                   // pieces of a row
    static constexpr int RP = CH >= 16 ? 1 : 16 / CH;                   // rows of 256 bytes, the width of the banks
    static constexpr int N = P * SLOTS * ROWS * CH;
    static constexpr int kBytes = N * 16;
    static constexpr int kPlane = SLOTS * ROWS * CH * 16;

    __device__ static __forceinline__ int swz(int row) { return (row / RP) & (CH - 1); }

    // Requests `left` rows from `at` (the first row of the tile's first head) straight into LDS: no registers, no waiting (AT_ARRIVE).  The
    // descriptor ends with the last of these rows and pieces beyond `dim` are addressed out of its range: both arrive as zeros.
    __device__ static __forceinline__ void request(const AtRows& src, const char* at, int dim, int left, unsigned lds) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), end = (left - 1) * (int)src.row + dim * 2;
#pragma unroll
        for (int n = 0; n < (N + kAtBlock - 1) / kAtBlock; ++n) {
            const int first = n * kAtBlock + wave * kWave;
            if (N % kAtBlock && first >= N) break;
            // (kAtBlock pieces are a whole number of a head's rows, or a head's rows are fewer: then two waves share one)
            const int ps = ROWS * CH >= kAtBlock ? n * kAtBlock / (CH * ROWS) : first / (CH * ROWS), slot = ps % SLOTS, plane = ps / SLOTS;
            const int row = (first + lane) / CH % ROWS, c = (lane % CH) ^ swz(row);
            const uint64_t base = (uint64_t)(uintptr_t)at + slot * src.head + plane * src.plane;
            const int voff = c * 8 < dim ? row * (int)src.row + c * 16 : (int)0x80000000;
            i32x4 rsrc = {(int)(uint32_t)base, (int)(uint32_t)((base >> 32) & 0xffffu), end, 0x00020000};
#pragma unroll
            for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
            lds_dma16(rsrc, __builtin_amdgcn_readfirstlane(lds + first * 16), voff, 0);
        }
    }

    // A lane's places in any tile, formed once: blocks, heads and planes are constant distances from them (the swizzle of rows 16 b + r is
    // that of r, and of rows 16 b + 4 g + r that of 4 g + r).
    struct Lane {
        int rows[DP / 32], turned[DP / 16];
        __device__ __forceinline__ Lane() {
            const int lane = lane_id(), i = lane & 15, g = lane >> 4, r = 4 * g + i / 4;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) rows[c] = (i * CH + ((4 * c + g) ^ swz(i))) * 16;
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) turned[b] = (r * CH + ((2 * b + (i % 4) / 2) ^ swz(r))) * 16 + (i & 1) * 8;
        }
    };
    // rows 16 b + (lane & 15), elements 32 c + 8 g ..: the A operand of a product over the elements
    __device__ static __forceinline__ Frag frag(const char* tile, const Lane& l, int slot, int b, int c) {
        const char* p = tile + (slot * ROWS + 16 * b) * CH * 16 + l.rows[c];
        if constexpr (P == 1) return *reinterpret_cast<const Frag*>(p);
        else {
            Frag f;
#pragma unroll
            for (int i = 0; i < P; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(p + i * kPlane);
            return f;
        }
    }
    // The A operand of a product over rows 32 j ..: elements 16 b + (lane & 15).  Sixteen lanes read four rows of sixteen elements, lane i
    // row i / 4 and elements 4 (i % 4) .., and receive element i of each row.
    __device__ static __forceinline__ i16x8 turned(const char* p) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(at_lds_t)p);
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(at_lds_t)(p + 16 * CH * 16));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    __device__ static __forceinline__ Frag frag_turned(const char* tile, const Lane& l, int slot, int j, int b) {
        const char* p = tile + (slot * ROWS + 32 * j) * CH * 16 + l.turned[b];
        if constexpr (P == 1) return __builtin_bit_cast(Frag, turned(p));
        else {
            Frag f;
#pragma unroll
            for (int i = 0; i < P; ++i) f.p[i] = __builtin_bit_cast(bf16x8, turned(p + i * kPlane));
            return f;
        }
    }
};

// every request of this wave has arrived and its LDS accesses are done; then the workgroup meets
#define AT_ARRIVE() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory")

// -- distance biases ----------------------------------------------------------------------------------------------------------------
// kSlope: -slope_h |c_i - c_j|.   kTable: table[bucket][h], bucket = number of edges (squared distances, ascending) <= |c_i - c_j|^2.
// The squared distance is a sum of squares of integers: exact in fp32 below 2^24, and every edge is at most 2^22.
// A bias enters a product as the accumulator it starts from, divided by the score's scale.
enum { kNone = 0, kSlope = 1, kTable = 2 };

// A bucket without a search: the leading bits of the fp32 squared distance (its octave and kCellBits bits behind) name a cell; a cell
// holds at most one edge (the host checks), so the bucket is the cell's first bucket, plus one behind that edge.  A cell is one word: the
// bucket in front in the low 8 bits, the edge's remaining bits above (beyond all of them: no edge).
constexpr int kCellBits = 5, kCellRest = 23 - kCellBits;
constexpr int kCellFirst = (127 << kCellBits) - 1;                        // 1.0 is cell 1; squared distance 0 is cell 0
constexpr int kCells = (22 << kCellBits) + 2;                             // 0, then [1, 2^22), then everything from 2^22 on

struct AtBias {
    const float* table;        // [buckets][heads]
    const unsigned* cells;     // [kCells]
    const float* slopes;       // [heads]
    int buckets;
};

// The cells and the table of HG heads as they stand in LDS: table[HG][kTableRow], already divided by the scale (neighbouring buckets in
// neighbouring banks), and cells whose bucket is a byte offset into a row (low 10 bits), so that a pair's one address serves every head.
constexpr int kTableRow = 64;
__device__ __forceinline__ void at_put_cells(unsigned* __restrict__ cells, const unsigned* __restrict__ src) {
    for (int i = threadIdx.x; i < kCells; i += kAtBlock) cells[i] = (src[i] >> 8 << 10) | (src[i] & 255u) * 4;
}
// A softmax only sees differences, and a score far enough below another is zero beside it.  So a head's finite entries keep their order and
// their differences up to 2^14 in units of log 2; what is farther apart counts as that far, and the largest is brought to at most 2^14: a row
// whose keys all carry the type's lowest value still has scores that differ and sums that fp32 resolves.  Entries within +-2^14 stay what
// they are.  A wave takes a head, a lane a bucket.
template <int HG>
__device__ __forceinline__ void at_put_table(float* __restrict__ table, const AtBias& bias, int heads, int h0, float scale) {
    const float most = 16384.f / kLog2e;
    const int lane = lane_id();
    for (int h = threadIdx.x >> 6; h < HG; h += kAtBlock / kWave) {
        float v = lane < bias.buckets ? bias.table[(int64_t)lane * heads + h0 + h] : INFINITY;
        const bool finite = fabsf(v) < INFINITY;
        if (__any(finite && fabsf(v) > most)) {
            auto largest = [&](bool of) {
                float m = of ? v : -INFINITY;
                for (int off = kWave / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
                return m;
            };
            // down the distinct values: `now` is what `at` becomes; from `top` on (as `put`) no two neighbours were too far apart
            float at = largest(finite), now = fminf(fmaxf(at, -most), most), top = at, put = now, mine = v;
            for (int n = 0; n < bias.buckets; ++n) {
                if (finite && v == at) mine = now;
                const float next = largest(finite && v < at);
                if (next == -INFINITY) break;
                if (at - next > most) {
                    top = next;
                    put = now = now - most;
                } else now = put == top ? next : put - (top - next);
                at = next;
            }
            v = mine;
        }
        if (lane < bias.buckets) table[h * kTableRow + lane] = v / scale;
    }
}
__device__ __forceinline__ int at_bucket(const unsigned* cells, float d2) {
    const int bits = __builtin_bit_cast(int, d2);
    const unsigned c = cells[min(max(bits >> kCellRest, kCellFirst), kCellFirst + kCells - 1) - kCellFirst];
    return (int)(c & 1023u) + ((unsigned)(bits & ((1 << kCellRest) - 1)) >= (c >> 10) ? 4 : 0);
}

// what the heads of a wave share about four pairs: distances, or their buckets' places in the table
template <int BIAS>
struct AtPairs {
    float d[4];
    int b[4];
    __device__ __forceinline__ void form(const float* cs, int rows, int at, float x, float y, float z, const unsigned* cells) {
        const f32x4 rx = *reinterpret_cast<const f32x4*>(cs + at), ry = *reinterpret_cast<const f32x4*>(cs + rows + at), rz = *reinterpret_cast<const f32x4*>(cs + 2 * rows + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float dx = rx[e] - x, dy = ry[e] - y, dz = rz[e] - z, d2 = dx * dx + dy * dy + dz * dz;
            if (BIAS == kSlope) d[e] = __builtin_amdgcn_sqrtf(d2);
            if (BIAS == kTable) b[e] = at_bucket(cells, d2);
        }
    }
    // the accumulator head h's block starts from
    __device__ __forceinline__ f32x4 start(float slope, const float* table, int h) const {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BIAS == kSlope) s[e] = slope * d[e];
            if (BIAS == kTable) s[e] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(table + h * kTableRow) + b[e]);
        }
        return s;
    }
};

inline const char* at_check(int64_t nseg, int64_t mq, int64_t mk, int heads, int kv_heads, int dim, int dtype, float scale, int mode, int buckets,
                            const int64_t* strides, int n_strides) {
    if (nseg < 1 || nseg > 1 << 20) return "need 1 <= segments <= 2^20";
    if (mq < 1 || mk < 0 || mq > 0x7fffffff - (1 << 22) || mk > 0x7fffffff - (1 << 22)) return "need 1 <= query rows, 0 <= key rows, both below 2^31 - 2^22";
    if (heads < 1 || heads > 1024 || kv_heads < 1 || heads % kv_heads) return "the key heads must divide the query heads (at most 1024)";
    if (mq * heads * 128 > (int64_t)1 << 33 || mk * kv_heads * 128 > (int64_t)1 << 33) return "need rows x heads <= 2^26";      // (one launch's workgroups)
    if (nseg * heads > 1 << 22) return "need segments x heads <= 2^22";                      // (likewise: a segment takes up to two workgroups a head)
    if (dim < 8 || dim > 128 || dim % 8) return "head dimension: a multiple of 8 in [8, 128]";
    if (dtype < 0 || dtype > 2) return "dtype: 0 fp32, 1 bf16, 2 fp16";
    if (!(scale >= 1e-6f && scale <= 1e6f)) return "need 1e-6 <= scale <= 1e6";
    if (mode < kNone || mode > kTable) return "bias: 0 none, 1 slopes, 2 table";
    if (mode == kTable && (buckets < 1 || buckets > 48)) return "need 1 <= buckets <= 48";
    for (int i = 0; i < n_strides; ++i)
        if (strides[i] < 0 || strides[i] % (dtype == 0 ? 4 : 8)) return "strides must be whole 16-byte pieces";
    for (int i = 0; i < n_strides; i += 2)
        if (strides[i] >= 1 << 22) return "a row stride must be below 2^22 elements";
    return nullptr;
}

// -- fp32 tensors as three bf16 planes [3][rows][heads][dim] -------------------------------------------------------------------------
inline int64_t at_plane_bytes(int64_t rows, int heads, int dim) { return rows * heads * dim * 2; }

static __global__ __launch_bounds__(256) void at_planes_kernel(const float* __restrict__ src, int64_t row_stride, int64_t head_stride, int64_t rows, int heads, int dim,
                                                              __bf16* __restrict__ out) {
    const int quads = dim / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = rows * heads * quads;
    if (i >= total) return;
    const int d = (int)(i % quads) * 4, h = (int)(i / quads % heads);
    const f32x4 v = *reinterpret_cast<const f32x4*>(src + i / quads / heads * row_stride + (int64_t)h * head_stride + d);
    bf16x4 p[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        __bf16 a, b, c;
        at_split(v[e], a, b, c);
        p[0][e] = a; p[1][e] = b; p[2][e] = c;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x4*>(out + ((int64_t)k * total + i) * 4) = p[k];
}

// the rows of a tensor as the kernels stream them: as they are, or (fp32) cut into planes at `planes`
template <typename T>
static AtRows at_stream(const void* p, int64_t row_stride, int64_t head_stride, int64_t rows, int heads, int dim, void* planes, hipStream_t st) {
    if constexpr (sizeof(T) == 4) {
        if (rows > 0)
            at_planes_kernel<<<(unsigned)ceil_div(rows * heads * (dim / 4), 256), 256, 0, st>>>((const float*)p, row_stride, head_stride, rows, heads, dim, (__bf16*)planes);
        return AtRows{(const char*)planes, (int64_t)heads * dim * 2, (int64_t)dim * 2, at_plane_bytes(rows, heads, dim)};
    }
    return AtRows{(const char*)p, row_stride * 2, head_stride * 2, 0};
}

}  // namespace lidiff
