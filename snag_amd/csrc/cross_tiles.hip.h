// Cross attention on the matrix pipe: what the tiled kernels share (csrc/cross_fwd.hip, csrc/cross_bwd.hip).
//
//   S = c2 q k^T (log2 domain),  p = exp2(S - lse),  o = p v;  dv = p^T do,  ds = p (do v^T - delta),  dq = scale ds k,  dk = scale ds^T q
//
// One wave owns 32 rows (forward, d q) or 32 keys (d k / d v) and keeps them as B operands of 32 x 32 products in its registers; the other
// side goes through LDS tiles that the workgroup's waves share.  The products are formed TRANSPOSED -- the owned index is the column, i.e.
// the lane -- so a softmax row is one lane pair: its maximum, sum and rescaling need one cross-lane exchange, and the probabilities leave
// the accumulators already in the B layout of the next product once the contraction index is taken in the accumulators' own order
// (keys 8 (i / 4) + 4 h + i % 4 for register i of lane half h); the A operand is read from LDS in that order (16 bit: transposing LDS reads).
// fp32 runs on the fp32 matrix instruction (32 x 32 x 2), so its sums and products are fp32 throughout; 16-bit inputs round p and ds to the
// inputs' type for the second products (what the matrix pipe takes); their sums, the running maximum and the row sums stay in fp32.
// fp16 keeps nothing below 2^-24, and the backward's operands are small: p is 1 / keys, ds about p |do| |v|.  They are rounded as 2^15 p and 2^e ds, e
// following the largest |ds| met so far (kHalfStart below); without that d q of 8192 keys
// was 7.5e-3 off for a d_out of 1e-3 and 7e-2 for 1e-4; now 9.6e-4 and 9.3e-3, which is the rounding of the fp16 result alone.  fp16 backwards take
// 2-7 % longer for it (2048 x 8192 x 128: 1066 -> 1106 us; heads of 100, whose d k / d v spills: 370 -> 427).
#pragma once
#include <type_traits>
#include "cross.hip.h"

namespace snag {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x8 = __attribute__((ext_vector_type(8))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
#if defined(__HIP_DEVICE_COMPILE__)
#define SNAG_LDS __attribute__((address_space(3)))
#define SNAG_GLOBAL __attribute__((address_space(1)))
#else
#define SNAG_LDS
#define SNAG_GLOBAL
#endif

// ---- LDS tiles: R rows of DP elements, without padding --------------------------------------------------------------------
// The 16-byte chunks of a row are permuted by the row.  LDS delivers 256 bytes a cycle, 16 lanes' chunks: the 16 rows that a fragment along the
// rows touches at a time, and the rows that one across them does (16 bit: four rows x four chunks a cycle; fp32: half a row each of rows r and
// r + 4), fall into different banks.  (fp32 rows of 32 elements, where two rows share the 256 bytes, keep a two-way conflict across.)
template <class T, int DP> __device__ __forceinline__ int chunk_place(int row, int chunk) {
    constexpr int bytes = DP * (int)sizeof(T);
    if constexpr (sizeof(T) == 4 && bytes >= 256) return chunk ^ ((((row >> 2) & 1) << 3) | (row & 3) | (((row >> 3) & 1) << 2));
    else if constexpr (bytes == 256) return chunk ^ (((row & 3) << 2) | ((row >> 2) & 3));
    else if constexpr (bytes == 128) return chunk ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
    else return chunk ^ ((row >> 2) & 3);
}
// place of element col (a multiple of the chunk) of a row
template <class T, int DP> __device__ __forceinline__ int tile_at(int row, int col) { return row * DP + chunk_place<T, DP>(row, col / Chunk<T>::n) * Chunk<T>::n; }

// ---- fragments: 16 contraction elements of 32 rows / columns, 8 per lane --------------------------------------------------
template <class T> struct Mma {
    using Frag = __attribute__((ext_vector_type(8))) T;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (std::is_same_v<T, bf16_t>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
#else
        return c;
#endif
    }
    // A operand whose contraction index runs along the LDS row: rows row0 .. row0 + 31, elements col0 + 8 h + j (row0: a multiple of 32)
    template <int DP> static __device__ __forceinline__ Frag rows(const T* base, int row0, int col0, int lane) {
        return *(const Frag*)(base + row0 * DP + tile_at<T, DP>(lane & 31, col0 + (lane >> 5) * 8));
    }
    // A operand whose contraction index runs over the LDS rows: columns col0 .. col0 + 31, LDS rows row0 + 8 (j / 4) + 4 h + j % 4 (row0: of 16).
    // The transposing read hands a group of 16 lanes a 4 x 16 block: lane t addresses row t / 4, columns 4 (t % 4), and receives column t.
    template <int DP> static __device__ __forceinline__ Frag cols(const T* base, int row0, int col0, int lane) {
        [[maybe_unused]] const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), c = col0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        union { Frag f; s16x4 h[2]; } u;
#if defined(__HIP_DEVICE_COMPILE__)
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)(base + row0 * DP + tile_at<T, DP>(r, c) + (c & 7)));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)(base + row0 * DP + tile_at<T, DP>(r + 8, c) + (c & 7)));
#endif
        return u.f;
    }
};
template <> struct Mma<float> {
    using Frag = f32x8;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
#endif
        return c;
    }
    template <int DP> static __device__ __forceinline__ Frag rows(const float* base, int row0, int col0, int lane) {
        const int c = col0 + (lane >> 5) * 8;
        const f32x4 a = *(const f32x4*)(base + row0 * DP + tile_at<float, DP>(lane & 31, c)), b = *(const f32x4*)(base + row0 * DP + tile_at<float, DP>(lane & 31, c + 4));
        return Frag{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    template <int DP> static __device__ __forceinline__ Frag cols(const float* base, int row0, int col0, int lane) {
        Frag f;
        const int c = col0 + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = base[row0 * DP + tile_at<float, DP>(4 * (lane >> 5) + 8 * (j >> 2) + (j & 3), c & ~3) + (c & 3)];
        return f;
    }
};

// accumulator registers 8 u .. 8 u + 7 (contraction block u of 16) as the B operand of the next product
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag pack(const f32x16& s, int u) {
    typename Mma<T>::Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)s[8 * u + j];
    return f;
}

// The power of two that fp16 operands ds carry.  It belongs to an output column, the lane pair's own row or key, so the accumulators carry it too and it
// is taken off when they are stored.  It starts at 2^60 (|ds| < 2^40: no overflow in fp32) and is lowered -- with the accumulators -- whenever a value passes 2^15,
// so that the largest lies in [2^8, 2^9): what is 2^-22 of it is still a normal number, and it takes a 64 times larger one to move the scale again.
constexpr float kHalfTop = 32768.f, kHalfStart = 60.f, kHalfP = 15.f;      // p <= 1 travels as 2^15 p
template <class T> constexpr bool kIsHalf = std::is_same_v<T, f16_t>;

// v of the other half of the wave (lane ^ 32), combined by the caller's operation
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
#else
    lo = hi = v;
#endif
}

// exponent by which the lane pair's power has to move (0 or less; infinities move nothing) for values whose largest magnitude is top
__device__ __forceinline__ int half_shift(float top) { return top > kHalfTop ? min(9 - __builtin_amdgcn_frexp_expf(top), 0) : 0; }
__device__ __forceinline__ float largest(const f32x16& s) {
    float a = 0.f, b = 0.f, lo, hi;
#pragma unroll
    for (int i = 0; i < 16; i += 2) a = fmaxf(a, fabsf(s[i])), b = fmaxf(b, fabsf(s[i + 1]));
    halves(fmaxf(a, b), lo, hi);
    return fmaxf(lo, hi);
}

// B operands of one row of d elements (the lane's own row), DP / 16 fragments of 8 elements
template <class T, int DP>
__device__ __forceinline__ void own_row(typename Mma<T>::Frag (&f)[DP / 16], const T* row, int d, bool valid, int vec, int lane) {
    constexpr int C = Chunk<T>::n;
    typename Chunk<T>::vec r[DP / 16 * 8 / C];
#pragma unroll
    for (int u = 0; u < DP / 16 * 8 / C; ++u) r[u] = load_raw<T>(row, (u / (8 / C)) * 16 + (lane >> 5) * 8 + u % (8 / C) * C, d, valid, vec);
#pragma unroll
    for (int u = 0; u < DP / 16 * 8 / C; ++u) {
        const auto c = fix_tail<T>(r[u], (u / (8 / C)) * 16 + (lane >> 5) * 8 + u % (8 / C) * C, d, vec);
#pragma unroll
        for (int j = 0; j < C; ++j) f[u / (8 / C)][u % (8 / C) * C + j] = c[j];
    }
}

// A tile of R rows on its way from global memory to LDS, one ahead of the tile that is worked on.  Every row pointer has to be readable.  What pads a
// tile has to be zeros when it is worked on: p is 0 there, but 0 x inf is NaN.
// DIRECT: straight into LDS, 16 bytes a lane, no registers; rows have to be whole (d == DP, 16-byte aligned).  pad() clears the rows from `count` on once the
// tile has landed (reading zeros in their place cost every tile 1-2 %).
// Otherwise through registers: on the way to LDS the columns behind d become zeros, and rows that are not to be kept do, whatever they hold.
// (Which rows those are is not known yet when the loads go out: nothing waits for a length or a mask.)
template <class T, int DP, int R, int NT, bool DIRECT>
struct TileFetch {
    static constexpr int C = Chunk<T>::n, kPerRow = DP / C, kAll = R * kPerRow, kN = (kAll + NT - 1) / NT;
    static_assert(kAll % NT == 0 || (kN == 1 && !DIRECT), "tile does not divide among the threads");
    typename Chunk<T>::vec r[DIRECT ? 1 : kN];
    template <class RowPtr>
    __device__ __forceinline__ void fetch(RowPtr row, T* lds, int d, int vec, int tid) {
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            const int e = u * NT + tid, i = e / kPerRow;
            if constexpr (DIRECT) {
                [[maybe_unused]] const T* p = row(i) + chunk_place<T, DP>(i, e % kPerRow) * C;
#if defined(__HIP_DEVICE_COMPILE__)
                __builtin_amdgcn_global_load_lds((SNAG_GLOBAL void*)p, (SNAG_LDS void*)(lds + (u * NT + (tid & ~63)) * C), 16, 0, 0);
#endif
            } else {
                const bool in = kAll % NT == 0 || e < kAll;
                r[u] = load_raw<T>(row(in ? i : 0), (e % kPerRow) * C, d, in, vec);
            }
        }
    }
    static __device__ __forceinline__ void pad(int count, T* lds, int tid) {
        if constexpr (DIRECT)
            for (int e = max(count, 0) * kPerRow + tid; e < kAll; e += NT) *(typename Chunk<T>::vec*)(lds + e * C) = typename Chunk<T>::vec{};
    }
    template <class Keep>
    __device__ __forceinline__ void store(Keep keep, T* lds, int d, int vec, int tid) const {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int u = 0; u < kN; ++u) {
                const int e = u * NT + tid, i = e / kPerRow;
                auto v = fix_tail<T>(r[u], (e % kPerRow) * C, d, vec);
                if (!keep(i)) v = typename Chunk<T>::vec{};
                if (kAll % NT == 0 || e < kAll) *(typename Chunk<T>::vec*)(lds + tile_at<T, DP>(i, (e % kPerRow) * C)) = v;
            }
        }
    }
};
// The tile in flight has landed, everybody's part of it, and everybody is done with the one before.
__device__ __forceinline__ void tile_ready() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// What this workgroup has written to LDS since is there for everybody.
__device__ __forceinline__ void pad_ready() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Writes a transposed accumulator (rows = elements, column = the lane's row): 4 neighbouring elements per register quad.
// lo (or NULL): the same place for what the rounding dropped.
template <class T, int DP>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DP / 32], float scale, int d, int lane, T* lo = nullptr) {
    const int h = lane >> 5;
    using V4 = __attribute__((ext_vector_type(4))) T;
    typedef V4 any4 __attribute__((aligned(sizeof(T))));
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = db * 32 + g * 8 + h * 4;
            V4 v, w;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (T)(acc[db][4 * g + j] * scale), w[j] = (T)(acc[db][4 * g + j] * scale - (float)v[j]);
            if (col + 4 <= d) {
                *(any4*)(row + col) = v;
                if (lo != nullptr) *(any4*)(lo + col) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < d) {
                        row[col + j] = v[j];
                        if (lo != nullptr) lo[col + j] = w[j];
                    }
            }
        }
}

struct Problem { int b, hk, split; int64_t tile; };
// workgroup -> (problem, split, tile): the tiles of one problem are neighbours, so that one XCD's L2 serves its keys
__device__ __forceinline__ Problem problem_of(const CrossArgs& a, int64_t tiles) {
    const uint32_t id = (uint32_t)xcd_order(blockIdx.x, gridDim.x), t = (uint32_t)tiles;      // fewer than 2^26 workgroups
    Problem p;
    p.tile = id % t;
    const uint32_t rest = id / t;
    p.split = (int)(rest % (uint32_t)a.splits);
    const uint32_t bh = rest / (uint32_t)a.splits;
    p.hk = (int)(bh % (uint32_t)a.Hkv);
    p.b = (int)(bh / (uint32_t)a.Hkv);
    return p;
}

__device__ __forceinline__ bool key_seen(const CrossArgs& a, int b, int key, int len) {
    return key < len && (a.mask == nullptr || a.mask[(int64_t)b * a.mask_ld + key] != 0);
}
// 64 keys from key0 as bits, one lane's look each
__device__ __forceinline__ bool mask_byte(const CrossArgs& a, int b, int key0, int lane) {
    return a.mask == nullptr || (key0 + lane < a.Lk && a.mask[(int64_t)b * a.mask_ld + key0 + lane] != 0);
}
__device__ __forceinline__ uint64_t seen_bits(bool byte, int key0, int len, int lane) { return __ballot(byte && key0 + lane < len); }
// -inf for the keys of a 32-key block that are not seen; bits: of the block
__device__ __forceinline__ void hide_keys(f32x16& s, uint32_t bits, int lane) {
    const uint32_t mine = bits >> (4 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1 ? s[i] : -INFINITY;
}
// row = l G + g: the host has checked that the multiplier is exact for every row
__device__ __forceinline__ int row_l(const CrossArgs& a, int row) { return (int)(__umulhi((uint32_t)row, a.g_magic) + ((uint32_t)row & a.g_one)); }

}  // namespace snag
