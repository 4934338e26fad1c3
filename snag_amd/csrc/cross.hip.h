// Cross attention: what its kernels share (csrc/cross_fwd.hip, csrc/cross_bwd.hip: tiles on the matrix pipe; csrc/cross_rows.hip: a few rows per key/value head;
// csrc/cross.hip: the choice between them).
//
// The rows of one problem (b, hk) are the Lq * G queries of the G = H / Hkv heads that share key/value head hk, row = l * G + g: a key/value
// tile is read once for all of them, and d K, d V of a shared head are sums inside one workgroup (no atomics).
#pragma once
#include <hip/hip_bf16.h>
#include "common.hip.h"

namespace snag {

using bf16_t = __bf16;
using f16_t = _Float16;
using f32x4 = __attribute__((ext_vector_type(4))) float;

struct CrossArgs {
    const void *q, *k, *v;
    int64_t qsb, qsl, qsh, ksb, ksl, ksh, vsb, vsl, vsh;      // element strides of batch / position / head; the head's own elements are adjacent
    int B, Lq, Lk, H, Hkv, G, d;
    int rows;                    // Lq * G
    uint32_t g_magic, g_one;     // row / G = high word of row * g_magic; G == 1: g_magic = 0, g_one = all ones
    const void* lens;            // [B] int32 / int64 or NULL: keys at and behind lens[b] are not seen
    int lens_bytes;
    const uint8_t* mask;         // [B, Lk] (row pitch mask_ld) or NULL: 0 = key not seen
    int64_t mask_ld;
    float scale, c2;             // c2 = scale * log2(e)
    int vec_q, vec_k, vec_v;     // 16-byte loads legal for this operand
    void *out, *out_lo;          // [B, Lq, H, d] dense; out_lo: what rounding to a 16-bit out dropped, or NULL
    float* lse;                  // [B, H, Lq]: log2 of the row's sum of exp2(c2 q.k); -inf for a row that sees no key
    int splits;                  // key ranges (forward, d q) or row ranges (d k, d v) worked on by different workgroups
    int per_split;               // keys / rows per range, a multiple of 64
    float* part;                 // splits > 1: partial results, see the kernels
    // backward
    const void *o, *o_lo, *dout; // [B, Lq, H, d] dense; o_lo or NULL
    float* stat;                 // [B, Hkv, padded_rows(rows)][2] = lse (+inf: no key seen), sum_d dout * o: d q writes it, d k / d v read it
    void *dq, *dk, *dv;          // dense, shapes of q, k, v
    int vec_o;                   // 16-byte access legal for the dense tensors (d a multiple of the chunk, aligned bases)
};

__device__ __forceinline__ int cross_len(const CrossArgs& a, int b) {
    if (a.lens == nullptr) return a.Lk;
    const int64_t n = a.lens_bytes == 4 ? (int64_t)((const int32_t*)a.lens)[b] : ((const int64_t*)a.lens)[b];
    return (int)(n < 0 ? 0 : (n > a.Lk ? a.Lk : n));
}

// Workgroup ids are dealt round-robin over the 8 XCDs: give neighbours in the logical order (the workgroups that read the same keys) one XCD's L2.
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t n) {
    const int64_t per = n >> 3;
    return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

template <class T> struct Chunk;                    // the 16 bytes a lane moves at once; `any`: the same at any address of an element
template <> struct Chunk<float> {
    static constexpr int n = 4;
    using vec = __attribute__((ext_vector_type(4))) float;
    typedef vec any __attribute__((aligned(4)));
};
template <> struct Chunk<bf16_t> {
    static constexpr int n = 8;
    using vec = __attribute__((ext_vector_type(8))) __bf16;
    typedef vec any __attribute__((aligned(2)));
};
template <> struct Chunk<f16_t> {
    static constexpr int n = 8;
    using vec = __attribute__((ext_vector_type(8))) _Float16;
    typedef vec any __attribute__((aligned(2)));
};

// Elements col .. col + n of a row of d elements; zero where the row is not valid or ends: load_raw, then -- where the value is used, so that the
// load can stay in flight until then -- fix_tail.  vec: d is a multiple of n and every row 16-byte aligned.  Otherwise rows take the same wide
// loads at any alignment; the chunk that the row's end cuts is loaded as the row's last n elements and shifted into place (element-wise loads
// made 4 heads of 75 fp16 elements three times slower).  Rows shorter than a chunk are loaded by element.
template <class T>
__device__ __forceinline__ typename Chunk<T>::vec load_raw(const T* __restrict__ row, int col, int d, bool valid, int vec) {
    constexpr int n = Chunk<T>::n;
    typename Chunk<T>::vec r{};
    if (valid && col < d) {
        if (vec) {
            r = *(const typename Chunk<T>::vec*)(row + col);
        } else if (d >= n) {
            r = *(const typename Chunk<T>::any*)(row + min(col, d - n));
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j)
                if (j < d) r[j] = row[j];
        }
    }
    return r;
}
template <class T>
__device__ __forceinline__ typename Chunk<T>::vec fix_tail(typename Chunk<T>::vec r, int col, int d, int vec) {
    constexpr int n = Chunk<T>::n;
    if (vec || d < n) return r;
    const int bits = max(col - (d - n), 0) * (int)sizeof(T) * 8;               // shift towards element 0
    union { typename Chunk<T>::vec v; uint64_t w[2]; } u{r};
    const uint64_t lo = bits < 64 ? (u.w[0] >> (bits & 63)) | ((u.w[1] << 1) << (63 - (bits & 63))) : u.w[1] >> (bits & 63);
    const uint64_t hi = u.w[1] >> (bits & 63);
    u.w[0] = bits < 128 ? lo : 0;
    u.w[1] = bits < 64 ? hi : 0;
    return u.v;
}
template <class T>
__device__ __forceinline__ typename Chunk<T>::vec load_chunk(const T* __restrict__ row, int col, int d, bool valid, int vec) {
    return fix_tail<T>(load_raw<T>(row, col, d, valid, vec), col, d, vec);
}

constexpr int64_t kLaunchWaves = ((int64_t)1 << 26) - 64;           // a launch has to stay below 2^32 threads

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// How a call is worked on (csrc/cross.hip chooses)
struct CrossPlan {
    int rows_path;               // a few rows per key/value head: csrc/cross_rows.hip
    int nw_fwd, nw_dq, nw_k;     // waves of a workgroup that owns rows (forward, d q) / keys
    int dp;                      // d rounded up to what the kernels are built for
    int s_fwd, s_dq, s_dkv;      // ranges
};
#define SNAG_CROSS_DP(CALL)                  \
    switch (p.dp) {                          \
        case 32: CALL(32); break;            \
        case 64: CALL(64); break;            \
        default: CALL(128); break;           \
    }

__host__ __device__ static inline int64_t padded_rows(int rows) { return ((int64_t)rows + 63) / 64 * 64; }
static inline int range_of(int n, int ranges) { return ((n + 63) / 64 + ranges - 1) / ranges * 64; }      // of n keys or rows

int cross_tiles_fwd(const CrossArgs& a, const CrossPlan& p, int dtype, hipStream_t st);
int cross_tiles_bwd(const CrossArgs& a, const CrossPlan& p, float* stat, int dtype, hipStream_t st);
int cross_combine(const CrossArgs& a, int dtype, hipStream_t st);
int cross_sum(const float* part, int64_t n, int ranges, void* out, int dtype, hipStream_t st);
int cross_rows_fwd(const CrossArgs& a, int dtype, hipStream_t st);
int cross_rows_bwd(const CrossArgs& a, int dtype, hipStream_t st);
int cross_rows_splits(int B, int Hkv, int Lk, int d, int dtype);

}  // namespace snag
