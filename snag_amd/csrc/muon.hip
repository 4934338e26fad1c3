// Newton-Schulz orthogonalisation of a list of matrices, alone or as the Muon update of their weights.
//
//   M <- mu M + (1 - mu) G,  U = nesterov ? (1 - mu) G + mu M : M          (step only; otherwise U = G)
//   X <- U / (|U|_F + eps)   as m x n, m <= n (a tall U enters transposed)
//   `steps` times:  A = X X^T,  B = b A + c A^2,  X <- a X + B X
//   W <- (1 - lr decay) W - lr s X                                         (step only; otherwise out = X)
//
// The products run on the matrix pipe in fp16 with fp32 accumulation.  fp16 keeps 11 bits, so every operand is stored as a pair (hi, lo) of
// fp16 values of ONE power-of-two scaling (X 2^14, A and B 2^13: |X| <= 1.21 and |A|, |B| <= 2.9 stay below fp16's 65504, and the small
// entries of a large matrix stay normal), 22 bits together:
//   * fp32 and fp16 matrices: three products hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of the product);
//   * bf16 matrices: one product hi hi, with the DIAGONALS of A and B kept out of it, in fp32:  with A = D + R,
//     A^2 = D^2 + D R + R D + R^2  and  a X + B X = (a + diag B) X + offdiag(B) X.  Near orthogonality A is almost its diagonal, and rounding
//     that diagonal to 11 bits is what dominates a plain fp16 iteration (2e-3 relative; 5e-4 this way, against 1.7e-3 for the rounding of
//     the bf16 result); the linear terms take R and X at 22 bits.
// A and B are symmetric: only tiles on and below the diagonal are computed, and both halves written.
// All matrices of the list share each launch.
#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>
#include "cross.hip.h"

namespace snag {

using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
#if defined(__HIP_DEVICE_COMPILE__)
#define SNAG_LDS __attribute__((address_space(3)))
#define SNAG_GLOBAL __attribute__((address_space(1)))
#else
#define SNAG_LDS
#define SNAG_GLOBAL
#endif

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kScaleX = 16384.f, kScaleA = 8192.f;
constexpr int kMaxList = 24;                   // matrices per launch (they travel as kernel arguments of the first one)
constexpr int kNormParts = 256;                // partial sums of |U|^2 per matrix

struct MuonMatrix {
    const void* g;
    float* mom;
    void* w;                 // step: the weight; otherwise the output
    char* work;              // this matrix's workspace
    int r, c, m, n, mp, np;  // shape; m <= n; both rounded up to whole tiles
    int tall;
    int cut[2], ranges[2];   // A (0) and A^2 (1): tiles from `cut` on are summed from `ranges` ranges of the contraction
    float update;            // lr * s
    int vec;                 // rows of g, mom and the result start 16-byte aligned
};
// What every launch needs, in device memory: kernel arguments lie in host memory, and a launch of a few workgroups spent most of its time on
// the chain of reads that finds its matrix (15 us for one tile).  The first launch of an update writes it.
struct MuonTable {
    int count, dtype, step, nesterov;
    float mu, keep, eps;     // keep = 1 - lr * decay
    int pad;
    MuonMatrix a[kMaxList];
};
static_assert(sizeof(MuonTable) <= 4096 && sizeof(MuonTable) % 16 == 0 && sizeof(MuonMatrix) % 8 == 0, "travels as kernel arguments");
constexpr int kTableBytes = 4096;

// workspace of one matrix
__host__ __device__ inline int64_t plane_x(const MuonMatrix& a) { return (int64_t)a.mp * a.np; }
__host__ __device__ inline int64_t plane_s(const MuonMatrix& a) { return (int64_t)a.mp * a.mp; }
// X in copy `k` (the iterations alternate), plane 0 = hi, 1 = lo
__device__ __forceinline__ _Float16* x_plane(const MuonMatrix& a, int k, int plane) { return (_Float16*)a.work + (2 * k + plane) * plane_x(a); }
// plane 0, 1: off-diagonal part of A; 2, 3: of B
__device__ __forceinline__ _Float16* s_plane(const MuonMatrix& a, int plane) { return (_Float16*)a.work + 4 * plane_x(a) + plane * plane_s(a); }
__device__ __forceinline__ double* norm_of(const MuonMatrix& a) { return (double*)((_Float16*)a.work + 4 * plane_x(a) + 4 * plane_s(a)); }
// diagonals of A (0) and B (1)
__device__ __forceinline__ float* diagonal(const MuonMatrix& a, int which) { return (float*)(norm_of(a) + kNormParts) + which * a.mp; }
__device__ __forceinline__ float* slab_of(const MuonMatrix& a) { return (float*)(norm_of(a) + kNormParts) + 2 * a.mp; }

template <int DT> using TypeOf = std::conditional_t<DT == SNAG_F32, float, std::conditional_t<DT == SNAG_BF16, bf16_t, f16_t>>;
template <class T> __device__ __forceinline__ float value(const void* p, int64_t i) { return (float)((const T*)p)[i]; }

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// ---- momentum and norm: grid (kNormParts, matrices) ----------------------------------------------------------------------
__device__ __forceinline__ float update_of(int nesterov, float mu, float g, float m) { return nesterov ? fmaf(1.f - mu, g, mu * m) : m; }

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void muon_norm_kernel(MuonTable L, MuonTable* __restrict__ table) {
    const MuonMatrix a = L.a[blockIdx.y];
    using T = TypeOf<DT>;
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        const int* src = (const int*)&L;
        for (int i = threadIdx.x; i < (int)(sizeof(MuonTable) / 4); i += 256) ((int*)table)[i] = src[i];
    }
    const int64_t n = (int64_t)a.r * a.c;
    double s = 0.0;                                // the norm of gradients of any size: fp32 squares would end at 1e19
    const int64_t step = (int64_t)gridDim.x * 256 * 4;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += step) {
        float u[4];
        if (VEC) {
            using V = __attribute__((ext_vector_type(4))) T;
            const V v = *(const V*)((const T*)a.g + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = (float)v[j];
            if (L.step) {
                f32x4 m = *(const f32x4*)(a.mom + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = fmaf(L.mu, m[j], (1.f - L.mu) * u[j]), u[j] = update_of(L.nesterov, L.mu, u[j], m[j]);
                *(f32x4*)(a.mom + i) = m;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = 0.f;
                if (i + j >= n) continue;
                u[j] = value<T>(a.g, i + j);
                if (L.step) {
                    const float m = fmaf(L.mu, a.mom[i + j], (1.f - L.mu) * u[j]);
                    a.mom[i + j] = m;
                    u[j] = update_of(L.nesterov, L.mu, u[j], m);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s += (double)u[j] * (double)u[j];
    }
    __shared__ double red[4];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) norm_of(a)[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// ---- X = U / (|U| + eps) as (hi, lo), padded with zeros: 64 x 64 blocks of X ----------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void muon_start_kernel(const MuonTable* __restrict__ L) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const MuonMatrix a = L->a[blockIdx.y];
    using T = TypeOf<DT>;
    const int step = L->step, nesterov = L->nesterov;
    const float mu = L->mu;
    const int cols = a.np / 64, blocks = (a.mp / 64) * cols;
    if ((int)blockIdx.x >= blocks) return;         // the whole workgroup
    double s = norm_of(a)[threadIdx.x];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]) + (double)L->eps;
    const double inv = (double)kScaleX / norm;     // beyond fp32's range for tiny gradients
    const int u = threadIdx.x >> 4, v = (threadIdx.x & 15) * 4;     // a thread's row (of 16 a turn) and first of its four columns
    _Float16 *xh = x_plane(a, 0, 0), *xl = x_plane(a, 0, 1);
    auto four = [&](int r, int c, float (&x)[4]) {                  // elements (r, c) .. (r, c + 3) of X, or of its transpose
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = 0.f;
        if (r >= a.r || c >= a.c) return;
        const int64_t at = (int64_t)r * a.c + c;
        if (a.vec) {                                                // c + 4 <= a.c: both are multiples of four
            using V = __attribute__((ext_vector_type(4))) T;
            const V g = *(const V*)((const T*)a.g + at);
            f32x4 m{};
            if (step) m = *(const f32x4*)(a.mom + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = step ? update_of(nesterov, mu, (float)g[j], m[j]) : (float)g[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < a.c) x[j] = step ? update_of(nesterov, mu, value<T>(a.g, at + j), a.mom[at + j]) : value<T>(a.g, at + j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)((double)x[j] * inv);
    };
    for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int i0 = blk / cols * 64, j0 = blk % cols * 64;       // rows and columns of X
        float x[4];
        if (a.tall) {
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 64; w += 16) {
                four(j0 + w + u, i0 + v, x);
#pragma unroll
                for (int j = 0; j < 4; ++j) tile[w + u][v + j] = x[j];
            }
            __syncthreads();
        }
#pragma unroll
        for (int w = 0; w < 64; w += 16) {
            if (a.tall) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = tile[v + j][w + u];
            } else {
                four(i0 + w + u, j0 + v, x);
            }
            f16x4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                _Float16 p, q;
                split16(x[j], p, q);
                hi[j] = p, lo[j] = q;
            }
            const int64_t at = (int64_t)(i0 + w + u) * a.np + j0 + v;
            *(f16x4*)(xh + at) = hi;
            *(f16x4*)(xl + at) = lo;
        }
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------
enum { kGram, kPoly, kApply };

// Workgroup shapes: a 128 x 128 tile by 4 waves of 64 x 64 (two stages: two workgroups a CU) or by 8 waves of 64 x 32 (four stages: one a CU, two
// waves a SIMD hide each other's waits), a 256 x 256 tile by 8 waves of 128 x 64.  64 / PLANES of the contraction per LDS stage, NST stages.
constexpr int threads_of(int tile, int nst) { return tile == 128 && nst == 2 ? 256 : 512; }
template <int TILE, int PLANES, int NST> struct Shape {
    static constexpr int kThreads = threads_of(TILE, NST), kWaves = kThreads / 64;
    static constexpr int kWm = TILE / 2, kWn = TILE * 2 / kWaves;      // a wave's part
    static constexpr int kDepth = 64 / PLANES, kChunks = kDepth / 8;   // 16-byte chunks per row of a stage
    static constexpr int kOperand = TILE * kDepth, kStage = 2 * PLANES * kOperand;     // fp16 values
    static constexpr int kLoads = kStage / 8 / kThreads;               // 16-byte loads of a thread per stage
    static constexpr size_t kLds = NST * kStage * sizeof(_Float16);
};

// Tile order: squares of 8 x 8 tiles one after another, so that the tiles that one XCD works on at a time share their operands in its L2.
constexpr int kSquare = 8;
__device__ __forceinline__ void tri_at(int k, int t, int& i, int& j) {     // tile k of those on and below the diagonal of t x t
    int I = 0, rows = min(kSquare, t);
    for (;;) {
        const int n = I * kSquare * rows + rows * (rows + 1) / 2;
        if (k < n) break;
        k -= n;
        ++I;
        rows = min(kSquare, t - I * kSquare);
    }
    const int J = k / (kSquare * rows);
    if (J < I) {
        k -= J * kSquare * rows;
        i = I * kSquare + k % rows;
        j = J * kSquare + k / rows;
    } else {
        k -= I * kSquare * rows;
        int q = 0;
        while ((q + 1) * (q + 2) / 2 <= k) ++q;
        i = I * kSquare + q;
        j = I * kSquare + k - q * (q + 1) / 2;
    }
}
__device__ __forceinline__ void rect_at(int k, int t, int u, int& i, int& j) {      // tile k of t x u
    const int J = k / (kSquare * t), cols = min(kSquare, u - J * kSquare);
    k -= J * kSquare * t;
    const int I = k / (kSquare * cols), rows = min(kSquare, t - I * kSquare);
    k -= I * kSquare * cols;
    i = I * kSquare + k % rows;
    j = J * kSquare + k / rows;
}

// First workgroup of every matrix in a launch (INT_MAX behind the list's end): a kernel argument, so that finding its matrix costs a workgroup no read
// of its own in front of the read of the matrix.
struct MuonFirst { int at[kMaxList]; };
__device__ __forceinline__ int matrix_of(const MuonFirst& first, int id, int& begin) {
    int which = 0;
    begin = first.at[0];
#pragma unroll
    for (int i = 1; i < kMaxList; ++i) which = id >= first.at[i] ? i : which, begin = id >= first.at[i] ? first.at[i] : begin;
    return __builtin_amdgcn_readfirstlane(which);
}

// one 16-byte chunk per lane straight from global memory into LDS: the wave's 64 chunks land at lds, in lane order
__device__ __forceinline__ void to_lds(const void* src, void* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds((SNAG_GLOBAL void*)src, (SNAG_LDS void*)lds, 16, 0, 0);
#endif
}

// LDS stage of a K-contiguous operand: [TILE rows][kDepth] fp16 with the chunks of a row permuted by the row.  LDS delivers 256 bytes a cycle, so
// the 16 rows that a fragment read touches at a time have to lie in different banks: rows of 128 bytes: chunk ^ row / 2 % 8, of 64 bytes:
// chunk ^ row / 4 % 4.
template <class S> __device__ __forceinline__ int place(int row, int chunk) { return S::kChunks == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3); }
template <class S, int TILE>
__device__ __forceinline__ void stage_rows(const _Float16* src, int ld, int row0, int k0, _Float16* lds, int wave, int lane) {
#pragma unroll
    for (int u = 0; u < TILE * S::kChunks / S::kThreads; ++u) {
        const int e = (u * S::kWaves + wave) * 64 + lane, r = e / S::kChunks, c = place<S>(r, e % S::kChunks);
        to_lds(src + (int64_t)(row0 + r) * ld + k0 + c * 8, lds + (u * S::kWaves + wave) * 512);
    }
}
template <class S>
__device__ __forceinline__ f16x8 frag_rows(const _Float16* lds, int row, int kb, int lane) {
    const int r = row + (lane & 31);
    return *(const f16x8*)(lds + r * S::kDepth + place<S>(lane & 31, kb * 2 + (lane >> 5)) * 8);       // row is a multiple of 32
}
// LDS stage of X as the right operand: [kDepth rows of the contraction][TILE columns], chunk c of row r at place c ^ 4 (r & 3): the four rows a
// transposing read takes from a 16-lane group lie in different banks.
template <class S, int TILE>
__device__ __forceinline__ void stage_cols(const _Float16* src, int ld, int k0, int col0, _Float16* lds, int wave, int lane) {
    constexpr int kRow = TILE / 8;
#pragma unroll
    for (int u = 0; u < TILE * S::kChunks / S::kThreads; ++u) {
        const int e = (u * S::kWaves + wave) * 64 + lane, r = e / kRow, c = (e % kRow) ^ ((r & 3) << 2);
        to_lds(src + (int64_t)(k0 + r) * ld + col0 + c * 8, lds + (u * S::kWaves + wave) * 512);
    }
}
template <int TILE>
__device__ __forceinline__ f16x8 frag_cols(const _Float16* lds, int col, int kb, int lane) {
    union { f16x8 f; s16x4 h[2]; } v;
    const int r = (lane >> 5) * 8 + ((lane & 15) >> 2), n = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    const int at = r * TILE + ((((col + n) >> 3) ^ ((r & 3) << 2)) * 8) + (n & 7) + kb * 16 * TILE;      // col is a multiple of 32
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int w = 0; w < 2; ++w) v.h[w] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)(lds + at + 4 * w * TILE));
#endif
    return v.f;
}

// 16 neighbouring fp16 pairs; as fp32 sums, and back
struct Pairs { f16x8 hi[2], lo[2]; };
__device__ __forceinline__ Pairs load_pairs(const _Float16* hi, const _Float16* lo) { return Pairs{{*(const f16x8*)hi, *(const f16x8*)(hi + 8)}, {*(const f16x8*)lo, *(const f16x8*)(lo + 8)}}; }
__device__ __forceinline__ float sum_of(const Pairs& p, int j) { return (float)p.hi[j >> 3][j & 7] + (float)p.lo[j >> 3][j & 7]; }
__device__ __forceinline__ Pairs pairs_of(const float (&v)[16]) {
    Pairs p;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        _Float16 x, y;
        split16(v[j], x, y);
        p.hi[j >> 3][j & 7] = x;
        p.lo[j >> 3][j & 7] = y;
    }
    return p;
}
__device__ __forceinline__ void store_pairs(_Float16* hi, _Float16* lo, const Pairs& p) {
    *(f16x8*)hi = p.hi[0], *(f16x8*)(hi + 8) = p.hi[1];
    *(f16x8*)lo = p.lo[0], *(f16x8*)(lo + 8) = p.lo[1];
}

// What a 32 x 32 block of the product becomes.  acc: register i of lane (h, l) = element (row0 + 8 (i / 4) + 4 h + i % 4, col0 + l).  The block goes
// through this wave's own piece of LDS (32 rows of kPitch floats, whole 16-byte steps), so that a lane holds 16 neighbours of one row and everything moves 16 bytes at
// a time; a tall result and the mirror image take 16 neighbours of one column instead.
constexpr int kPitch = 36;
// LDS keeps a wave's accesses in order; this keeps the compiler from moving one lane's reads in front of another's writes
__device__ __forceinline__ void lds_turn() { asm volatile("" ::: "memory"); }
// what a block needs of memory: X (APPLY) or the off-diagonal part of A (POLY) where it lies
template <int MODE>
__device__ __forceinline__ Pairs block_pairs(const MuonMatrix& a, int row0, int col0, int from, int lane) {
    const int row = row0 + (lane >> 1), col = col0 + (lane & 1) * 16;
    if (MODE == kApply) return load_pairs(x_plane(a, from, 0) + (int64_t)row * a.np + col, x_plane(a, from, 1) + (int64_t)row * a.np + col);
    if (MODE == kPoly) return load_pairs(s_plane(a, 0) + (int64_t)row * a.mp + col, s_plane(a, 1) + (int64_t)row * a.mp + col);
    return Pairs{};
}
// the accumulators through LDS: lane (r, c) gets columns c .. c + 15 of row r
__device__ __forceinline__ void through_block(float* block, const f32x16& acc, float (&v)[16], int lane) {
    const int h = lane >> 5, r = lane >> 1, c = (lane & 1) * 16;
    lds_turn();
#pragma unroll
    for (int i = 0; i < 16; ++i) block[(8 * (i >> 2) + 4 * h + (i & 3)) * kPitch + (lane & 31)] = acc[i];
    lds_turn();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 x = *(const f32x4*)(block + r * kPitch + c + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j];
    }
}
// values of 16 neighbours of a row become 16 neighbours of a column: lane (r, c) gets rows c .. c + 15 of column r
__device__ __forceinline__ void turn(float* block, float (&v)[16], int r, int c) {
    lds_turn();
#pragma unroll
    for (int q = 0; q < 4; ++q) *(f32x4*)(block + r * kPitch + c + 4 * q) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    lds_turn();
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = block[(c + j) * kPitch + r];
}
// element `at` (0 .. 15, else nothing) of v: its value; set to 0
__device__ __forceinline__ void clear(float (&v)[16], int at) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = j == at ? 0.f : v[j];
}
__device__ __forceinline__ float pick(const float (&v)[16], int at) {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) x = j == at ? v[j] : x;
    return x;
}
// the last iteration's 16 values of X (row, col ..; times 2^14) into the user's matrix
template <class T>
__device__ __forceinline__ void store_result(const MuonTable* __restrict__ L, const MuonMatrix& a, float (&v)[16], int row0, int col0, float* block, int lane) {
    const int r = lane >> 1, c = (lane & 1) * 16;
    int i0 = row0 + r, j0 = col0 + c;                      // where they go: row i0, columns j0 ..
    if (a.tall) {
        turn(block, v, r, c);
        i0 = col0 + r;
        j0 = row0 + c;
    }
    if (i0 >= a.r || j0 >= a.c) return;
    T* out = (T*)a.w + (int64_t)i0 * a.c + j0;
    using V = typename Chunk<T>::vec;
    constexpr int C = Chunk<T>::n;
    const int step = L->step;
    const float keep = L->keep;
    if (j0 + 16 <= a.c && a.vec) {
#pragma unroll
        for (int q = 0; q < 16 / C; ++q) {
            V o;
            if (step) o = *(const V*)(out + q * C);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float x = v[q * C + j] * (1.f / kScaleX);
                o[j] = (T)(step ? fmaf(-a.update, x, keep * (float)o[j]) : x);
            }
            *(V*)(out + q * C) = o;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j0 + j >= a.c) continue;
            const float x = v[j] * (1.f / kScaleX);
            out[j] = (T)(step ? fmaf(-a.update, x, keep * (float)out[j]) : x);
        }
    }
}

// B from A: v in: A^2's off-diagonal share times 2^26, out: B without its diagonal times 2^13; p: A's off-diagonal part; -> B's diagonal where `at` is on it
// (on: the block has a piece of the diagonal)
__device__ __forceinline__ float poly(float (&v)[16], const Pairs& p, float di, const float (&dj)[16], int at, bool on) {
    const float sq = on ? pick(v, at) * (1.f / (kScaleA * kScaleA)) : 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = fmaf(fmaf(kNsC, di + dj[j], kNsB), sum_of(p, j), v[j] * (kNsC / kScaleA));
    if (on) clear(v, at);
    return fmaf(kNsB, di, kNsC * fmaf(di, di, sq));
}
__device__ __forceinline__ void load16(float (&v)[16], const float* p) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 x = *(const f32x4*)(p + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = x[j];
    }
}

// the diagonals a block needs: of its row (APPLY: B's, POLY: A's), and of its columns (POLY)
struct Diagonals { float row, col[16]; };
template <int MODE>
__device__ __forceinline__ Diagonals block_diagonals(const MuonMatrix& a, int row0, int col0, int lane) {
    Diagonals d{};
    if (MODE != kGram) d.row = diagonal(a, MODE == kApply ? 1 : 0)[row0 + (lane >> 1)];
    if (MODE == kPoly) load16(d.col, diagonal(a, 0) + col0 + (lane & 1) * 16);
    return d;
}

template <int MODE, int DT>
__device__ __forceinline__ void finish(const MuonTable* __restrict__ L, const MuonMatrix& a, const f32x16& acc, const Pairs& p, const Diagonals& g, int row0, int col0, bool mirror, int from, bool last,
                                       float* block, int lane) {
    const int r = lane >> 1, c = (lane & 1) * 16;                          // row r, columns c .. c + 15 of the block
    const int row = row0 + r, col = col0 + c, at = row - col;
    float v[16];
    through_block(block, acc, v, lane);
    if constexpr (MODE == kApply) {
        const float d = kNsA + g.row;
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = fmaf(d, sum_of(p, j), v[j] * (1.f / kScaleA));                                 // times 2^14
        if (last) store_result<TypeOf<DT>>(L, a, v, row0, col0, block, lane);
        else store_pairs(x_plane(a, from ^ 1, 0) + (int64_t)row * a.np + col, x_plane(a, from ^ 1, 1) + (int64_t)row * a.np + col, pairs_of(v));
    } else {
        _Float16 *oh = s_plane(a, MODE == kGram ? 0 : 2), *ol = s_plane(a, MODE == kGram ? 1 : 3);
        float d;
        if constexpr (MODE == kGram) {
            d = pick(v, at) * (1.f / (kScaleX * kScaleX));
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] *= kScaleA / (kScaleX * kScaleX);
            if (row0 == col0) clear(v, at);
        } else {
            d = poly(v, p, g.row, g.col, at, row0 == col0);
        }
        if (at >= 0 && at < 16) diagonal(a, MODE == kGram ? 0 : 1)[row] = d;
        store_pairs(oh + (int64_t)row * a.mp + col, ol + (int64_t)row * a.mp + col, pairs_of(v));
        if (mirror) {
            turn(block, v, r, c);
            const int64_t to = (int64_t)(col0 + r) * a.mp + row0 + c;
            store_pairs(oh + to, ol + to, pairs_of(v));
        }
    }
}

// PLANES 1: hi hi, 2: hi hi + hi lo + lo hi.  The LDS stages are filled straight from memory, NST - 1 ahead; the fragments of the next 16 of the
// contraction are read while the present ones are multiplied, across the stages too: the barrier that opens a stage stands in front of the
// last products of the stage before it.
// 4096 x 4096 in bf16: A 91 - 94 us (0.75 - 0.78 PFLOP/s), A^2 93 - 95, B X 155 - 177 (0.78 - 0.89); a library product of that size: 110 (1.24).
template <int MODE, int DT, int TILE, int NST>
__global__ __launch_bounds__(threads_of(TILE, NST), 2) void muon_product_kernel(const MuonTable* __restrict__ L, MuonFirst first, int whole, int from, int last) {
    constexpr int PLANES = DT == SNAG_BF16 ? 1 : 2;
    using S = Shape<TILE, PLANES, NST>;
    constexpr int NI = S::kWm / 32, NJ = S::kWn / 32, KB = S::kDepth / 16;
    static_assert(KB % 2 == 0, "fragment sets alternate");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16* lds = (_Float16*)smem;
    const int lane = threadIdx.x & 63, wave = wave_id_uniform();
    // ranges of cut tiles have a launch's last ids, and are dealt over the XCDs as they come
    const int id = (int)blockIdx.x < whole ? (int)xcd_order(blockIdx.x, whole) : (int)blockIdx.x;
    int begin;
    const MuonMatrix a = L->a[matrix_of(first, id, begin)];
    int k = id - begin, split = 0, ti, tj;
    bool cut = false;
    if (MODE == kApply) {
        rect_at(k, a.mp / TILE, a.np / TILE, ti, tj);
    } else {
        const int t = a.mp / TILE, c0 = a.cut[MODE];
        cut = k >= c0;
        if (cut) {
            const int n = t * (t + 1) / 2 - c0;
            split = (k - c0) / n;
            k = c0 + (k - c0) % n;
        }
        tri_at(k, t, ti, tj);
    }
    const int lda = MODE == kGram ? a.np : a.mp;
    int k0 = 0, k1 = lda;
    if (MODE != kApply && cut) {
        const int per = (lda / 64 + a.ranges[MODE] - 1) / a.ranges[MODE] * 64;
        k0 = split * per;
        k1 = min(lda, k0 + per);
    }
    const int n = k1 > k0 ? (k1 - k0) / S::kDepth : 0;                 // stages
    const _Float16* left = MODE == kGram ? x_plane(a, from, 0) : s_plane(a, MODE == kPoly ? 0 : 2);
    const _Float16* right = MODE == kPoly ? left : x_plane(a, from, 0);
    const int64_t left_lo = MODE == kGram ? plane_x(a) : plane_s(a), right_lo = MODE == kPoly ? plane_s(a) : plane_x(a);
    auto stage = [&](int t) {
        const int kk = k0 + t * S::kDepth;
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
            _Float16* base = lds + t % NST * S::kStage + q * 2 * S::kOperand;
            stage_rows<S, TILE>(left + q * left_lo, lda, ti * TILE, kk, base, wave, lane);
            if (MODE == kApply) stage_cols<S, TILE>(right + q * right_lo, a.np, kk, tj * TILE, base + S::kOperand, wave, lane);
            else stage_rows<S, TILE>(right + q * right_lo, lda, tj * TILE, kk, base + S::kOperand, wave, lane);
        }
    };
    f32x16 acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x16{};
    constexpr int kWavesN = TILE / S::kWn;
    const int wm = (wave / kWavesN) * S::kWm, wn = (wave % kWavesN) * S::kWn;
    // A launch of one workgroup per CU takes its blocks' own values along with the first stages; otherwise they are fetched one block ahead.
    Pairs own[NI * NJ];
    Diagonals diag[NI * NJ];
    const int i0 = ti * TILE + wm, j0 = tj * TILE + wn;
    auto fetch = [&](int q) {
        own[q] = block_pairs<MODE>(a, i0 + q / NJ * 32, j0 + q % NJ * 32, from, lane);
        diag[q] = block_diagonals<MODE>(a, i0 + q / NJ * 32, j0 + q % NJ * 32, lane);
    };
    if (NST > 2) {
#pragma unroll
        for (int q = 0; q < NI * NJ; ++q) fetch(q);
    }
    f16x8 fa[2][PLANES][NI], fb[2][PLANES][NJ];
    auto read = [&](int set, int t, int kb) {
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
            const _Float16* o = lds + t % NST * S::kStage + q * 2 * S::kOperand;
#pragma unroll
            for (int i = 0; i < NI; ++i) fa[set][q][i] = frag_rows<S>(o, wm + i * 32, kb, lane);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[set][q][j] = MODE == kApply ? frag_cols<TILE>(o + S::kOperand, wn + j * 32, kb, lane) : frag_rows<S>(o + S::kOperand, wn + j * 32, kb, lane);
        }
    };
    // stage t has landed, everybody's part of it, and everybody is done reading the one before it.  Loads in flight: of stages t .. t + NST - 2
    auto open = [&](int t) {
        if (NST > 2 && t + NST - 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * S::kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (n > 0) {
#pragma unroll
        for (int t = 0; t < NST - 1; ++t)
            if (t < n) stage(t);
        open(0);
        if (NST - 1 < n) stage(NST - 1);
        read(0, 0, 0);
    }
    for (int t = 0; t < n; ++t) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if (kb + 1 < KB) {
                read((kb + 1) & 1, t, kb + 1);
            } else if (t + 1 < n) {
                open(t + 1);
                if (t + NST < n) stage(t + NST);
                read(0, t + 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            const int set = kb & 1;
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][0][i], fb[set][0][j], acc[i][j], 0, 0, 0);
                    if constexpr (PLANES == 2) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][0][i], fb[set][1][j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][1][i], fb[set][0][j], acc[i][j], 0, 0, 0);
                    }
                }
#endif
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (MODE != kApply && cut) {
        // the range's partial tile, 32 x 32 blocks in register order: muon_sum_kernel adds the ranges up
        const int t = a.mp / TILE, c0 = a.cut[MODE], n = t * (t + 1) / 2 - c0;
        float* out = slab_of(a) + (int64_t)(split * n + k - c0) * 16 * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) *(f32x16*)(out + ((wm / 32 + i) * 4 + wn / 32 + j) * 1024) = acc[i][j];
        return;
    }
    __syncthreads();                                           // the stages become the waves' blocks
    float* block = (float*)smem + wave * 32 * kPitch;
    if (NST == 2) fetch(0);
#pragma unroll
    for (int q = 0; q < NI * NJ; ++q) {
        if (NST == 2 && q + 1 < NI * NJ) fetch(q + 1);
        finish<MODE, DT>(L, a, acc[q / NJ][q % NJ], own[q], diag[q], i0 + q / NJ * 32, j0 + q % NJ * 32, ti != tj, from, last != 0, block, lane);
    }
}

// The cut tiles of A or A^2 from their ranges: a workgroup per 32 x 32 block of the 128 x 128 tiles, each of its four waves adds up a quarter of the ranges, in order; the
// quarters are joined through LDS (eight waves: 10 us instead of 6 for six matrices around 1024 x 1024).  Grid (16 x the largest number of cut tiles, matrices)
template <int MODE>
__global__ __launch_bounds__(256) void muon_sum_kernel(const MuonTable* __restrict__ L) {
    __shared__ float block[32 * kPitch];
    __shared__ __attribute__((aligned(16))) f32x16 part[3][64];
    const MuonMatrix a = L->a[blockIdx.y];
    const int t = a.mp / 128, tiles = t * (t + 1) / 2 - a.cut[MODE], id = blockIdx.x >> 4, sub = blockIdx.x & 15, lane = threadIdx.x & 63, quarter = wave_id_uniform();
    if (id >= tiles) return;     // the whole workgroup
    const int per = (a.ranges[MODE] + 3) / 4, s1 = min(a.ranges[MODE], (quarter + 1) * per);
    int s = quarter * per;
    f32x16 acc{};
    const int64_t step = (int64_t)tiles * 16 * 1024;
    const float* p = slab_of(a) + ((int64_t)id * 16 + sub) * 1024 + lane * 16 + s * step;
    for (; s + 8 <= s1; s += 8, p += 8 * step) {
        f32x16 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = *(const f32x16*)(p + u * step);
#pragma unroll
        for (int u = 0; u < 8; ++u) acc += v[u];
    }
    for (; s < s1; ++s, p += step) acc += *(const f32x16*)p;
    if (quarter > 0) part[quarter - 1][lane] = acc;
    __syncthreads();
    if (quarter > 0) return;
#pragma unroll
    for (int u = 0; u < 3; ++u) acc += part[u][lane];
    int i, j;
    tri_at(a.cut[MODE] + id, t, i, j);
    const int row0 = i * 128 + (sub >> 2) * 32, col0 = j * 128 + (sub & 3) * 32;
    finish<MODE, SNAG_F32>(L, a, acc, block_pairs<MODE>(a, row0, col0, 0, lane), block_diagonals<MODE>(a, row0, col0, lane), row0, col0, i != j, 0, false, block, lane);
}

// ---- one side of at most 128 ------------------------------------------------------------------------------------------------
// A is one 128 x 128 tile: every workgroup of a 64-column block of X computes B for itself, in LDS, and goes on to its block of the new X and
// that block's share of the next A.  An iteration is two launches (this one and muon_sum_kernel, which adds the shares up) in place of
// four, and these matrices are all latency: 128 x 128 .. 128 x 4096, 22 launches of 6-14 us before, 13 now.  Eight waves, two a SIMD, of 64 x 32 (A^2,
// the shares) and 32 x 32 (B X) hide each other's waits (128 x 128 .. 128 x 4096 in fp32: 14.7 us a launch; 17.9 with 128 columns and four waves).
// LDS images: [128 rows][128] fp16 with chunk c (16 bytes) of row r at place c ^ (4 (r % 4) + r / 4 % 4), and X's block [128 rows][64] with chunk c at
// c ^ (4 (r / 2 % 2) + r / 4 % 4): without bank conflicts both for fragments along the rows and for transposing reads across them.
constexpr int kBlock = 64;                                             // columns of X per workgroup
template <int COLS> struct Image {
    static constexpr int kSize = 128 * COLS, kChunks = COLS / 8;
    static __device__ __forceinline__ int turn(int row) { return COLS == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }
    static __device__ __forceinline__ int at(int row, int col) { return row * COLS + (((col >> 3) ^ turn(row)) << 3) + (col & 7); }
    static __device__ __forceinline__ void load(const _Float16* src, int ld, _Float16* lds, int wave, int lane) {
#pragma unroll
        for (int u = 0; u < kSize / 8 / 512; ++u) {
            const int e = (u * 8 + wave) * 64 + lane, r = e / kChunks, c = e % kChunks ^ turn(r);
            to_lds(src + (int64_t)r * ld + c * 8, lds + (u * 8 + wave) * 512);
        }
    }
    static __device__ __forceinline__ f16x8 rows(const _Float16* lds, int row, int kb, int lane) { return *(const f16x8*)(lds + at(row + (lane & 31), kb * 16 + (lane >> 5) * 8)); }
    static __device__ __forceinline__ f16x8 cols(const _Float16* lds, int col, int kb, int lane) {
        union { f16x8 f; s16x4 h[2]; } v;
        [[maybe_unused]] const int r = kb * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2), n = col + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int w = 0; w < 2; ++w) v.h[w] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)(lds + at(r + 4 * w, n)));
#endif
        return v.f;
    }
    static __device__ __forceinline__ Pairs pairs(const _Float16* lds, int row, int col) {
        const _Float16* lo = lds + kSize;
        return Pairs{{*(const f16x8*)(lds + at(row, col)), *(const f16x8*)(lds + at(row, col + 8))}, {*(const f16x8*)(lo + at(row, col)), *(const f16x8*)(lo + at(row, col + 8))}};
    }
    static __device__ __forceinline__ void store(_Float16* lds, int row, int col, const Pairs& p) {
        _Float16* lo = lds + kSize;
        *(f16x8*)(lds + at(row, col)) = p.hi[0], *(f16x8*)(lds + at(row, col + 8)) = p.hi[1];
        *(f16x8*)(lo + at(row, col)) = p.lo[0], *(f16x8*)(lo + at(row, col + 8)) = p.lo[1];
    }
};
// NB blocks of 32 x 32 below each other over 16 KB of the contraction: left(plane, block, kb) and right(plane, kb) are the fragments.  The next 16 of the
// contraction are read while the present ones are multiplied.
template <int PLANES, int NB, int KB, class Left, class Right>
__device__ __forceinline__ void image_product(f32x16 (&acc)[NB], Left left, Right right) {
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = f32x16{};
    f16x8 fa[2][PLANES][NB], fb[2][PLANES];
    auto read = [&](int kb) {
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
#pragma unroll
            for (int i = 0; i < NB; ++i) fa[kb & 1][p][i] = left(p, i, kb);
            fb[kb & 1][p] = right(p, kb);
        }
    };
    read(0);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        if (kb + 1 < KB) read(kb + 1);
        __builtin_amdgcn_sched_barrier(0);
        [[maybe_unused]] const int s = kb & 1;
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][0][i], fb[s][0], acc[i], 0, 0, 0);
            if constexpr (PLANES == 2) {
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][0][i], fb[s][1], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][1][i], fb[s][0], acc[i], 0, 0, 0);
            }
        }
#endif
        __builtin_amdgcn_sched_barrier(0);
    }
}

// start: only the first A's shares of X copy 0.  One workgroup per 64-column block; slab[block][4][4][1024] as the product kernel's ranges.
template <int DT>
__global__ __launch_bounds__(512) void muon_narrow_kernel(const MuonTable* __restrict__ L, MuonFirst first, int from, int start, int last) {
    constexpr int PLANES = DT == SNAG_BF16 ? 1 : 2;
    using IX = Image<kBlock>;
    using IS = Image<128>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16 *X = (_Float16*)smem, *S = X + 2 * IX::kSize;             // hi, lo of X's block; hi, lo of A, later of B
    float* diag = (float*)(S + 2 * IS::kSize);                         // B's diagonal [128], and behind it the waves' 32 x kPitch blocks
    const int lane = threadIdx.x & 63, wave = wave_id_uniform();
    float* block = diag + 128 + wave * 32 * kPitch;
    int begin;
    const MuonMatrix a = L->a[matrix_of(first, blockIdx.x, begin)];
    const int col0 = ((int)blockIdx.x - begin) * kBlock;
    const int wm = (wave >> 2) * 64, wn = (wave & 3) * 32;             // 64 x 32 of A, B
    const int xm = (wave >> 1) * 32, xn = (wave & 1) * 32;             // 32 x 32 of X's block
    IX::load(x_plane(a, from, 0) + col0, a.np, X, wave, lane);
    IX::load(x_plane(a, from, 1) + col0, a.np, X + IX::kSize, wave, lane);
    f32x16 acc[2];
    const int r = lane >> 1, c = (lane & 1) * 16;
    if (!start) {
        IS::load(s_plane(a, 0), 128, S, wave, lane);
        IS::load(s_plane(a, 1), 128, S + IS::kSize, wave, lane);
        const float* da = diagonal(a, 0);
        float di[2], dj[16];
#pragma unroll
        for (int i = 0; i < 2; ++i) di[i] = da[wm + i * 32 + r];
        load16(dj, da + wn + c);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        image_product<PLANES, 2, 8>(acc, [&](int p, int i, int kb) { return IS::rows(S + p * IS::kSize, wm + i * 32, kb, lane); },
                                    [&](int p, int kb) { return IS::rows(S + p * IS::kSize, wn, kb, lane); });
        // B in the place of A
        Pairs b[2];
        float db[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = wm + i * 32 + r, col = wn + c;
            const Pairs p = IS::pairs(S, row, col);
            float v[16];
            through_block(block, acc[i], v, lane);
            db[i] = poly(v, p, di[i], dj, row - col, wm + i * 32 == wn);
            b[i] = pairs_of(v);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = wm + i * 32 + r, col = wn + c;
            IS::store(S, row, col, b[i]);
            if (row >= col && row < col + 16) diag[row] = db[i];
        }
        __syncthreads();
        f32x16 bx[1];
        image_product<PLANES, 1, 8>(bx, [&](int p, int, int kb) { return IS::rows(S + p * IS::kSize, xm, kb, lane); },
                                    [&](int p, int kb) { return IX::cols(X + p * IX::kSize, xn, kb, lane); });
        const int row = xm + r, col = xn + c;
        const Pairs p = IX::pairs(X, row, col);
        float v[16];
        through_block(block, bx[0], v, lane);
        const float d = kNsA + diag[row];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = fmaf(d, sum_of(p, j), v[j] * (1.f / kScaleA));
        if (last) {
            store_result<TypeOf<DT>>(L, a, v, xm, col0 + xn, block, lane);
            return;
        }
        const Pairs y = pairs_of(v);
        const int64_t at = (int64_t)row * a.np + col0 + col;
        store_pairs(x_plane(a, from ^ 1, 0) + at, x_plane(a, from ^ 1, 1) + at, y);
        __syncthreads();
        IX::store(X, row, col, y);
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
    image_product<PLANES, 2, kBlock / 16>(acc, [&](int p, int i, int kb) { return IX::rows(X + p * IX::kSize, wm + i * 32, kb, lane); },
                                          [&](int p, int kb) { return IX::rows(X + p * IX::kSize, wn, kb, lane); });
    if (a.ranges[kGram] == 1) {                                        // the only block: A is complete
#pragma unroll
        for (int i = 0; i < 2; ++i) finish<kGram, DT>(L, a, acc[i], Pairs{}, Diagonals{}, wm + i * 32, wn, false, 0, false, block, lane);
        return;
    }
    float* out = slab_of(a) + (int64_t)(col0 / kBlock) * 16 * 1024 + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) *(f32x16*)(out + ((wm / 32 + i) * 4 + wn / 32) * 1024) = acc[i];
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static int pad_to(int n, int tile) { return (n + tile - 1) / tile * tile; }
constexpr int kCus = 256;

// How one list of matrices is worked on.  narrow: every m <= 128 (muon_narrow_kernel).  Otherwise the product with X takes the tiles whose rounds are done
// first: 512 tiles of 128 x 128 run at a time (two a CU), or 256 of 256 x 256, four times the work, which read half as much per multiplication and take 3-6 % less
// than two rounds of small ones.  bf16, large / small tiles: 8 matrices of 1024 x 1024 (one round / one) 541 / 477 us, 9 of them (one / two) 539 / 546, 2816 x 2816
// (one / one) 861 / 702, 3584 x 3584 (one / two) 1321 / 1393, 4352 x 4352 (two / three) 2814 / 2509.  The symmetric products, half as many tiles, always run on
// 128 x 128 ones.
struct MuonPlan { bool narrow; int tile, stages, over, over_ranges[2]; };
static int pad_n(const MuonPlan& p, int n) { return pad_to(n, p.narrow ? kBlock : p.tile); }
static int splits_of(const MuonPlan& p, int np) { return p.narrow ? np / kBlock : (np / 64 + p.stages - 1) / p.stages; }
static MuonPlan plan_of(const int32_t* rows, const int32_t* cols, const int* at, int count) {
    MuonPlan p{};
    p.narrow = true, p.tile = 128;
    int64_t big = 0, small = 0, total = 0;
    for (int k = 0; k < count; ++k) {
        const int r = rows[at[k]], c = cols[at[k]], m = r < c ? r : c, n = r < c ? c : r;
        p.narrow = p.narrow && m <= 128;
        big += (int64_t)(pad_to(m, 256) / 256) * (pad_to(n, 256) / 256);
        const int64_t t = pad_to(m, 128) / 128;
        small += t * (pad_to(n, 128) / 128);
        total += t * (t + 1) / 2 * (pad_to(n, 128) / 64);
    }
    if (!p.narrow && 2 * ((big + kCus - 1) / kCus) <= (small + 2 * kCus - 1) / (2 * kCus)) p.tile = 256;
    // LDS stages in a range of A's contraction: the list's stages over all CUs, at least four
    const int64_t per = (total + kCus - 1) / kCus;
    p.stages = (int)(per < 4 ? 4 : per);
    // The symmetric products run 512 tiles at a time.  A few tiles more (up to 128) would be a round of their own on an empty chip: the last tiles of the
    // last matrix, the list's largest, are cut into ranges of at least eight stages that fill it (4096 x 4096 in bf16, 16 tiles over: 116 -> 91 us and 5 for muon_sum_kernel).
    if (p.narrow) return p;
    int64_t tiles = 0;
    bool split = false;
    for (int k = 0; k < count; ++k) {
        const int r = rows[at[k]], c = cols[at[k]], t = pad_to(r < c ? r : c, p.tile) / 128;
        tiles += t * (t + 1) / 2;
        split = split || splits_of(p, pad_n(p, r < c ? c : r)) > 1;
    }
    const int r = rows[at[count - 1]], c = cols[at[count - 1]], mp = pad_to(r < c ? r : c, p.tile), np = pad_n(p, r < c ? c : r), t = mp / 128;
    const int over = (int)(tiles % (2 * kCus));
    if (split || tiles < 2 * kCus || over == 0 || over > kCus / 2 || over > t * (t + 1) / 2 || mp < 64 * 16) return p;
    p.over = over;
    for (int q = 0; q < 2; ++q) {
        const int most = (q ? mp : np) / 64 / 8, want = 2 * kCus / over;
        p.over_ranges[q] = most < want ? most : want;
    }
    return p;
}

// where the cut tiles of matrix `r` x `c` begin and how many ranges each has, for A and A^2
static void cuts_of(const MuonPlan& p, int mp, int np, bool last, int (&cut)[2], int (&ranges)[2]) {
    const int t = mp / 128, tiles = t * (t + 1) / 2, s = splits_of(p, np);
    for (int q = 0; q < 2; ++q) {
        ranges[q] = last && p.over > 0 ? p.over_ranges[q] : q == 0 ? s : 1;
        cut[q] = last && p.over > 0 ? tiles - p.over : ranges[q] > 1 ? 0 : tiles;
    }
}
static int64_t matrix_bytes(const MuonPlan& p, int r, int c, bool last) {
    const int m = r < c ? r : c, n = r < c ? c : r, mp = pad_to(m, p.tile), np = pad_n(p, n), t = mp / 128;
    int cut[2], ranges[2];
    cuts_of(p, mp, np, last, cut, ranges);
    int64_t slab = 0;                                              // 128 x 128 partial tiles: A's, then A^2's
    for (int q = 0; q < 2; ++q) slab = std::max(slab, (int64_t)ranges[q] * (t * (t + 1) / 2 - cut[q]));
    const int64_t x = (int64_t)mp * np, q = (int64_t)mp * mp;
    const int64_t bytes = 8 * x + 8 * q + 8 * kNormParts + 8 * (int64_t)mp + 4 * slab * 128 * 128;
    return (bytes + 255) / 256 * 256;
}

// A call's matrices in the order they are worked on: the narrow ones first, kMaxList at a time.
struct MuonLists {
    const int32_t *rows, *cols;
    int count, pass = 0, i = 0, n = 0, at[kMaxList];
    MuonLists(const int32_t* r, const int32_t* c, int k) : rows(r), cols(c), count(k) {}
    bool next() {                                              // the next list in at[0 .. n)
        for (n = 0; pass < 2; ++pass, i = 0) {
            for (; i < count && n < kMaxList; ++i)
                if (((rows[i] < cols[i] ? rows[i] : cols[i]) <= 128) == (pass == 0)) at[n++] = i;
            if (n > 0) {
                int big = 0;                                   // the largest goes last
                auto side = [&](int k) { return rows[at[k]] < cols[at[k]] ? rows[at[k]] : cols[at[k]]; };
                for (int k = 1; k < n; ++k) big = side(k) > side(big) ? k : big;
                std::swap(at[big], at[n - 1]);
                return true;
            }
        }
        return false;
    }
};

struct MuonRun { MuonTable L; MuonFirst first[3]; MuonTable* table; MuonPlan plan; int blocks_of[3], cut_tiles[2], blocks; bool vec; };

// more than 64 KB of LDS for `kernel`, once per device (done: a bit each; devices from 64 on are set every time)
template <class K>
static int grow_lds(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && dev < 64 && (done.load() >> dev & 1)) return SNAG_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return fail(SNAG_ERR_LAUNCH, "muon: %s", hipGetErrorString(e));
    if (dev < 64) done.fetch_or((uint64_t)1 << dev);
    return SNAG_OK;
}
template <int MODE, int DT, int TILE, int NST>
static int product_of(const MuonRun& R, int from, int last, hipStream_t st) {
    using S = Shape<TILE, DT == SNAG_BF16 ? 1 : 2, NST>;
    static std::atomic<uint64_t> done{0};
    if (int rc = grow_lds(muon_product_kernel<MODE, DT, TILE, NST>, S::kLds, done)) return rc;
    int whole = R.blocks_of[MODE];                             // tiles before the ranges of cut ones (a list all of whose matrices are cut: in any order)
    if (MODE != kApply && R.plan.over > 0) whole -= R.plan.over * R.plan.over_ranges[MODE];
    muon_product_kernel<MODE, DT, TILE, NST><<<dim3(R.blocks_of[MODE]), S::kThreads, S::kLds, st>>>(R.table, R.first[MODE], whole, from, last);
    return check_launch("muon_product");
}
// A 128 x 128 workgroup takes 64 KB of LDS with two stages, so that two fit a CU and hide each other's waits; a launch with at most one per CU
// takes 128 KB and loads three stages ahead instead.
template <int MODE, int DT>
static int product(const MuonRun& R, int from, int last, hipStream_t st) {
    if constexpr (MODE == kApply) {
        if (R.plan.tile == 256) return product_of<MODE, DT, 256, 2>(R, from, last, st);
    }
    if (R.blocks_of[MODE] <= kCus) return product_of<MODE, DT, 128, 4>(R, from, last, st);
    return product_of<MODE, DT, 128, 2>(R, from, last, st);
}

template <int MODE>
static int sum(const MuonRun& R, hipStream_t st) {
    if (R.cut_tiles[MODE] == 0) return SNAG_OK;
    muon_sum_kernel<MODE><<<dim3(16 * R.cut_tiles[MODE], R.L.count), 256, 0, st>>>(R.table);
    return check_launch("muon_sum");
}

template <int DT>
static int muon_go(const MuonRun& R, int steps, hipStream_t st) {
    const dim3 gn(kNormParts, R.L.count), gs(R.blocks < 2048 ? R.blocks : 2048, R.L.count);
    if (R.vec) muon_norm_kernel<DT, true><<<gn, 256, 0, st>>>(R.L, R.table);
    else muon_norm_kernel<DT, false><<<gn, 256, 0, st>>>(R.L, R.table);
    if (int rc = check_launch("muon_norm")) return rc;
    muon_start_kernel<DT><<<gs, 256, 0, st>>>(R.table);
    if (int rc = check_launch("muon_start")) return rc;
    if (R.plan.narrow) {
        constexpr size_t lds = 2 * (Image<kBlock>::kSize + Image<128>::kSize) * sizeof(_Float16) + (8 * 32 * kPitch + 128) * sizeof(float);
        static_assert(lds <= 160 * 1024, "one CU's LDS");
        static std::atomic<uint64_t> done{0};
        if (int rc = grow_lds(muon_narrow_kernel<DT>, lds, done)) return rc;
        for (int k = -1; k < steps; ++k) {
            if (k >= 0)
                if (int rc = sum<kGram>(R, st)) return rc;
            muon_narrow_kernel<DT><<<dim3(R.blocks_of[kApply]), 512, lds, st>>>(R.table, R.first[kApply], k < 0 ? 0 : k & 1, k < 0, k + 1 == steps);
            if (int rc = check_launch("muon_narrow")) return rc;
        }
        return SNAG_OK;
    }
    for (int k = 0; k < steps; ++k) {
        if (int rc = product<kGram, DT>(R, k & 1, 0, st)) return rc;
        if (int rc = sum<kGram>(R, st)) return rc;
        if (int rc = product<kPoly, DT>(R, k & 1, 0, st)) return rc;
        if (int rc = sum<kPoly>(R, st)) return rc;
        if (int rc = product<kApply, DT>(R, k & 1, k + 1 == steps, st)) return rc;
    }
    return SNAG_OK;
}

static int muon_check(const char* what, const int32_t* rows, const int32_t* cols, int count, int dtype) {
    SNAG_REQUIRE(dtype == SNAG_F32 || dtype == SNAG_BF16 || dtype == SNAG_F16, SNAG_ERR_ARG, "%s: dtype %d", what, dtype);
    SNAG_REQUIRE(count >= 0 && (count == 0 || (rows != nullptr && cols != nullptr)), SNAG_ERR_ARG, "%s: %d matrices, null shapes", what, count);
    for (int i = 0; i < count; ++i) {
        SNAG_REQUIRE(rows[i] >= 1 && cols[i] >= 1, SNAG_ERR_ARG, "%s: matrix %d is %d x %d", what, i, rows[i], cols[i]);
        SNAG_REQUIRE(rows[i] <= SNAG_MUON_MAX_SIDE && cols[i] <= SNAG_MUON_MAX_SIDE, SNAG_ERR_UNSUPPORTED, "%s: matrix %d is %d x %d: a side is longer than %d", what, i, rows[i], cols[i],
                     SNAG_MUON_MAX_SIDE);
    }
    return SNAG_OK;
}

static int64_t work_bytes_of(const int32_t* rows, const int32_t* cols, int count) {
    int64_t most = 0;
    for (MuonLists o(rows, cols, count); o.next();) {
        const MuonPlan p = plan_of(rows, cols, o.at, o.n);
        int64_t bytes = kTableBytes;
        for (int i = 0; i < o.n; ++i) bytes += matrix_bytes(p, rows[o.at[i]], cols[o.at[i]], i + 1 == o.n);
        most = bytes > most ? bytes : most;
    }
    return most;
}

// All matrices of a call; every list of launches starts at the workspace's beginning (they follow each other on the stream).
static int muon_run(const char* what, void* const* w, const void* const* g, float* const* mom, const int32_t* rows, const int32_t* cols, int count, int dtype, float lr, float mu, int nesterov,
                    float decay, int match_rms, int steps, float eps, void* work, int64_t work_bytes, void* stream) {
    if (int rc = muon_check(what, rows, cols, count, dtype)) return rc;
    SNAG_REQUIRE(steps >= 1 && steps <= 100, SNAG_ERR_ARG, "%s: %d steps", what, steps);
    SNAG_REQUIRE(eps >= 0.f, SNAG_ERR_ARG, "%s: eps %g", what, (double)eps);
    if (count == 0) return SNAG_OK;
    SNAG_REQUIRE(w != nullptr && g != nullptr, SNAG_ERR_ARG, "%s: null pointer lists", what);
    for (int i = 0; i < count; ++i) SNAG_REQUIRE(w[i] != nullptr && g[i] != nullptr && (mom == nullptr || mom[i] != nullptr), SNAG_ERR_ARG, "%s: null matrix %d", what, i);
    const int64_t need = work_bytes_of(rows, cols, count);
    SNAG_REQUIRE(work != nullptr && ((uintptr_t)work & 255) == 0 && work_bytes >= need, SNAG_ERR_ARG, "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)work_bytes,
                 (long long)need);
    for (MuonLists o(rows, cols, count); o.next();) {
        const int *at = o.at, n = o.n;
        MuonRun R{};
        R.plan = plan_of(rows, cols, at, n);
        const int tile = R.plan.tile;
        MuonTable& L = R.L;
        L.count = n;
        L.dtype = dtype, L.step = mom != nullptr, L.nesterov = nesterov, L.mu = mu, L.keep = 1.f - lr * decay, L.eps = eps;
        R.table = (MuonTable*)work, R.vec = true;
        for (auto& f : R.first)
            for (int& at0 : f.at) at0 = INT32_MAX;
        char* space = (char*)work + kTableBytes;
        for (int i = 0; i < n; ++i) {
            MuonMatrix& a = L.a[i];
            const int r = rows[at[i]], c = cols[at[i]];
            a.g = g[at[i]], a.w = w[at[i]], a.mom = mom != nullptr ? mom[at[i]] : nullptr, a.work = space;
            a.r = r, a.c = c, a.tall = r > c, a.m = r < c ? r : c, a.n = r < c ? c : r;
            a.mp = pad_to(a.m, tile), a.np = pad_n(R.plan, a.n);
            cuts_of(R.plan, a.mp, a.np, i + 1 == n, a.cut, a.ranges);
            const double s = match_rms ? 0.2 * sqrt((double)a.n) : sqrt(r > c ? (double)r / c : 1.0);
            a.update = (float)(lr * s);
            a.vec = c % 8 == 0 && aligned16(a.g) && aligned16(a.mom) && aligned16(a.w);
            space += matrix_bytes(R.plan, r, c, i + 1 == n);
            const int t = a.mp / 128, tri = t * (t + 1) / 2, b = (a.mp / 64) * (a.np / 64);
            for (int q = 0; q < 3; ++q) R.first[q].at[i] = R.blocks_of[q];
            for (int q = 0; q < 2; ++q) {
                R.blocks_of[q] += a.cut[q] + (tri - a.cut[q]) * a.ranges[q];
                R.cut_tiles[q] = std::max(R.cut_tiles[q], tri - a.cut[q]);
            }
            R.blocks_of[kApply] += R.plan.narrow ? a.np / kBlock : (a.mp / tile) * (a.np / tile);
            R.blocks = b > R.blocks ? b : R.blocks;
            R.vec = R.vec && (int64_t)r * c % 4 == 0 && aligned16(a.g) && aligned16(a.mom);
        }
        hipStream_t st = (hipStream_t)stream;
        if (int rc = dtype == SNAG_F32 ? muon_go<SNAG_F32>(R, steps, st) : dtype == SNAG_BF16 ? muon_go<SNAG_BF16>(R, steps, st) : muon_go<SNAG_F16>(R, steps, st)) return rc;
    }
    return SNAG_OK;
}

}  // namespace snag

using namespace snag;

extern "C" SNAG_API int64_t snag_muon_work_bytes(const int32_t* rows_host, const int32_t* cols_host, int count) {
    if (rows_host == nullptr || cols_host == nullptr) return 0;
    for (int i = 0; i < count; ++i)                        // refused by the call itself
        if (rows_host[i] < 1 || cols_host[i] < 1 || rows_host[i] > SNAG_MUON_MAX_SIDE || cols_host[i] > SNAG_MUON_MAX_SIDE) return 0;
    return work_bytes_of(rows_host, cols_host, count);
}

extern "C" SNAG_API int snag_orthogonalize(const void* const* g_host, void* const* out_host, const int32_t* rows_host, const int32_t* cols_host, int count, int dtype,
                                           int steps, float eps, void* work, int64_t work_bytes, void* stream) {
    return muon_run("orthogonalize", out_host, g_host, nullptr, rows_host, cols_host, count, dtype, 0.f, 0.f, 0, 0.f, 0, steps, eps, work, work_bytes, stream);
}

extern "C" SNAG_API int snag_muon_step(void* const* w_host, const void* const* g_host, float* const* momentum_host, const int32_t* rows_host, const int32_t* cols_host,
                                       int count, int dtype, float lr, float momentum, int nesterov, float weight_decay, int match_rms, int steps, float eps,
                                       void* work, int64_t work_bytes, void* stream) {
    SNAG_REQUIRE(count <= 0 || momentum_host != nullptr, SNAG_ERR_ARG, "muon step: null momentum list");
    SNAG_REQUIRE(momentum >= 0.f && momentum < 1.f, SNAG_ERR_ARG, "muon step: momentum %g is not in [0, 1)", (double)momentum);
    return muon_run("muon step", w_host, g_host, momentum_host, rows_host, cols_host, count, dtype, lr, momentum, nesterov, weight_decay, match_rms, steps, eps, work, work_bytes, stream);
}
