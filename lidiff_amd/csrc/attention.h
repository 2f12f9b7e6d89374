// Pieces shared by the attention kernels (attention_fwd.hip, attention_bwd.hip): element types, matrix products, distance biases,
// row tiles in LDS.
//
// One wave owns 16 "columns" (queries, or keys in the dK / dV kernel) of HG heads at a time and walks over tiles of 64 "rows" of the
// other side.  A product S = X Y^T with 16 x 16 blocks of v_mfma_f32_16x16x32 leaves in lane l the column l & 15 and the rows
// 4 (l >> 4) .. + 3 of a block: a column's statistics live in its own lanes, and the block IS (after rounding to the operands' type) half
// of the B operand of the next product over the rows -- no value crosses a lane.  A contraction may take its terms in any order as long
// as both operands agree, so rows 32 j + 16 (e / 4) + 4 g + e % 4 are the terms 8 g + e of lane group g of product j.
#pragma once
#include "segments.h"

namespace lidiff {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
struct alignas(16) f32x8 { f32x4 lo, hi; };

constexpr int kAtBlock = 256;      // 4 waves
constexpr int kAtRows = 64;        // rows of a tile
constexpr float kLog2e = 1.44269504088896340736f;

template <typename T> struct AtType;
template <> struct AtType<__bf16> { typedef bf16x8 Frag; typedef bf16x4 Quad; static constexpr int kPad = 8; static constexpr int kLift = 0, kPieces = 2; };
template <> struct AtType<_Float16> { typedef f16x8 Frag; typedef f16x4 Quad; static constexpr int kPad = 8; static constexpr int kLift = 15, kPieces = 2; };
template <> struct AtType<float> { typedef f32x8 Frag; typedef f32x4 Quad; static constexpr int kPad = 4; static constexpr int kLift = 0, kPieces = 1; };
// kLift: fp16 ends at 2^-24, where a probability of a long scan may well lie: probabilities are multiplied by 2^15 (at most 32768) before
// they are rounded to an fp16 operand, and the sums by 2^-15 -- exact, and an addend of the exponent that is there anyway.

// acc += A B over 32 terms: lane group g = lane >> 4 holds the terms 8 g .. 8 g + 7 of row (A) / column (B) lane & 15
__device__ __forceinline__ void at_mma(f32x4& acc, const bf16x8& a, const bf16x8& b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void at_mma(f32x4& acc, const f16x8& a, const f16x8& b) { acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ void at_mma(f32x4& acc, const f32x8& a, const f32x8& b) {      // eight products of four terms, one of each lane group
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], acc, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], acc, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ typename AtType<T>::Frag at_zero() {
    return typename AtType<T>::Frag{};
}

// eight consecutive elements (16 or 32 bytes)
template <typename T>
__device__ __forceinline__ typename AtType<T>::Frag at_frag(const T* p) {
    return *reinterpret_cast<const typename AtType<T>::Frag*>(p);
}
template <>
__device__ __forceinline__ f32x8 at_frag<float>(const float* p) {
    return f32x8{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)};
}

// a fragment of a transposed tile: four consecutive rows, and the four rows 16 further
template <typename T>
__device__ __forceinline__ typename AtType<T>::Frag at_frag_rows(const T* p) {
    typedef typename AtType<T>::Quad Quad;
    const Quad lo = *reinterpret_cast<const Quad*>(p), hi = *reinterpret_cast<const Quad*>(p + 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <>
__device__ __forceinline__ f32x8 at_frag_rows<float>(const float* p) {
    return f32x8{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 16)};
}

// two accumulator blocks (rows 32 j .. + 15 and + 16 .. + 31) as the B operand of the next product.  For 16-bit operands this rounds the
// probabilities (or their gradients) once, to the type the other operand has: the matrix instruction takes one type.
__device__ __forceinline__ void at_pack(bf16x8& f, const f32x4& a, const f32x4& b) {
    typedef float f32x8v __attribute__((ext_vector_type(8)));
    const f32x8v v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    f = __builtin_convertvector(v, bf16x8);
}
__device__ __forceinline__ void at_pack(f16x8& f, const f32x4& a, const f32x4& b) {
    typedef float f32x8v __attribute__((ext_vector_type(8)));
    const f32x8v v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    f = __builtin_convertvector(v, f16x8);
}
__device__ __forceinline__ void at_pack(f32x8& f, const f32x4& a, const f32x4& b) { f = f32x8{a, b}; }

// what the rounding of at_pack left (a, b: the values on entry, what is still left on return), as a second operand: two pieces carry 16
// (bf16) or 22 (fp16) bits; a third one changed the table gradient of 3 10^8 pairs by nothing (1.19e-6 against 1.18e-6)
template <typename F>
__device__ __forceinline__ void at_pack_rest(F& rest, const F& piece, f32x4& a, f32x4& b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] -= (float)piece[e]; b[e] -= (float)piece[4 + e]; }
    at_pack(rest, a, b);
}

// four consecutive outputs
template <typename T>
__device__ __forceinline__ void at_store4(T* p, const f32x4& v) {
    typedef typename AtType<T>::Quad Quad;
    *reinterpret_cast<Quad*>(p) = __builtin_convertvector(v, Quad);
}

// -- distance biases ----------------------------------------------------------------------------------------------------------------
// kSlope: -slope_h |c_i - c_j|.   kTable: table[bucket][h], bucket = number of edges (squared distances, ascending) <= |c_i - c_j|^2.
// The squared distance is a sum of squares of integers: exact in fp32 below 2^24, and every edge is at most 2^22.
enum { kNone = 0, kSlope = 1, kTable = 2 };

// A bucket without a search: the leading bits of the fp32 squared distance (its octave and kCellBits bits behind) name a cell; a cell
// holds at most one edge (the host checks), so the bucket is the cell's first bucket, plus one behind that edge.
constexpr int kCellBits = 5;
constexpr int kCellFirst = 127 << kCellBits;                              // cell of 1.0; squared distance 0 shares the cell in front
constexpr int kCells = (22 << kCellBits) + 2;                             // 0, then [1, 2^22), then everything from 2^22 on
struct alignas(8) AtCell { float edge; int bucket; };

__device__ __forceinline__ int at_cell(float d2) {
    const int c = (__builtin_bit_cast(int, d2) >> (23 - kCellBits)) - (kCellFirst - 1);
    return min(max(c, 0), kCells - 1);
}

struct AtBias {
    const float* table;        // [buckets][H]
    const AtCell* cells;       // [kCells]
    const float* slopes;       // [H]
    int buckets;
};

// tiles in LDS: [slot][64][DP + pad] rows as they are, [slot][DP][64 + 4] transposed
template <typename T, int DP>
struct AtTile {
    static constexpr int kRow = DP + AtType<T>::kPad;
    static constexpr int kCol = kAtRows + 4;
    static constexpr int kRows = kAtRows * kRow;
    static constexpr int kCols = DP * kCol;
};

// rows [lo, lo + 64) of `src` (element strides row / head, first head h0) into registers: 16 bytes a piece, kPieces a thread
template <typename T, int DP, int SLOTS>
struct AtLoad {
    static constexpr int kVec = 16 / (int)sizeof(T);
    static constexpr int kPerRow = DP / kVec;                          // pieces of a (row, head)
    static constexpr int kPieces = kAtRows * SLOTS * kPerRow / kAtBlock;
    static_assert(kAtRows * SLOTS * kPerRow % kAtBlock == 0, "whole pieces per thread");
    f32x4 r[kPieces];

    __device__ __forceinline__ static void place(int p, int& row, int& slot, int& d) {
        const int i = p * kAtBlock + threadIdx.x;
        d = (i % kPerRow) * kVec;
        slot = (i / kPerRow) % SLOTS;
        row = i / (kPerRow * SLOTS);
    }
    __device__ __forceinline__ void fetch(const T* __restrict__ src, int64_t row_stride, int64_t head_stride, int h0, int dim, int lo, int hi) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            int row, slot, d;
            place(p, row, slot, d);
            r[p] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (lo + row < hi && d < dim) r[p] = *reinterpret_cast<const f32x4*>(src + (int64_t)(lo + row) * row_stride + (int64_t)(h0 + slot) * head_stride + d);
        }
    }
    __device__ __forceinline__ void put_rows(T* __restrict__ dst) const {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            int row, slot, d;
            place(p, row, slot, d);
            *reinterpret_cast<f32x4*>(dst + slot * AtTile<T, DP>::kRows + row * AtTile<T, DP>::kRow + d) = r[p];
        }
    }
    __device__ __forceinline__ void put_cols(T* __restrict__ dst) const {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            int row, slot, d;
            place(p, row, slot, d);
            union { f32x4 v; T e[kVec]; } u;
            u.v = r[p];
#pragma unroll
            for (int e = 0; e < kVec; ++e) dst[slot * AtTile<T, DP>::kCols + (d + e) * AtTile<T, DP>::kCol + row] = u.e[e];
        }
    }
};

}  // namespace lidiff

namespace lidiff {

// Heads of one wave: the distances of a (query, key) pair are the same for every head, so with a distance bias a wave takes as many heads
// as the LDS tiles hold (4 x 32 or 2 x 64 elements); they have to be whole groups of one key head, or all have key heads of their own.
inline int at_heads_per_wave(int dim, int heads, int share, int mode) {
    const int n = dim <= 32 ? 4 : dim <= 64 ? 2 : 1;
    return mode != kNone && heads % n == 0 && (share == 1 || share % n == 0) ? n : 1;
}

inline const char* at_check(int64_t nseg, int64_t mq, int64_t mk, int heads, int kv_heads, int dim, int dtype, int mode, int buckets, const int64_t* strides,
                            int n_strides) {
    if (nseg < 1 || nseg > 1 << 20) return "need 1 <= segments <= 2^20";
    if (mq < 1 || mk < 0 || mq > 0x7fffffff - (1 << 22) || mk > 0x7fffffff - (1 << 22)) return "need 1 <= query rows, 0 <= key rows, both below 2^31 - 2^22";
    if (heads < 1 || heads > 1024 || kv_heads < 1 || heads % kv_heads) return "the key heads must divide the query heads (at most 1024)";
    if (dim < 8 || dim > 128 || dim % 8) return "head dimension: a multiple of 8 in [8, 128]";
    if (dtype < 0 || dtype > 2) return "dtype: 0 fp32, 1 bf16, 2 fp16";
    if (mode < kNone || mode > kTable) return "bias: 0 none, 1 slopes, 2 table";
    if (mode == kTable && (buckets < 1 || buckets > 48)) return "need 1 <= buckets <= 48";
    for (int i = 0; i < n_strides; ++i)
        if (strides[i] < 0 || strides[i] % (dtype == 0 ? 4 : 8)) return "strides must be whole 16-byte pieces";
    return nullptr;
}

}  // namespace lidiff
