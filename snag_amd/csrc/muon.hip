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
//   * fp32 matrices: three products hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of the product);
//   * 16-bit matrices: one product hi hi, with the DIAGONALS of A and B kept out of it, in fp32:  with A = D + R,
//     A^2 = D^2 + D R + R D + R^2  and  a X + B X = (a + diag B) X + offdiag(B) X.  Near orthogonality A is almost its diagonal, and rounding
//     that diagonal to 11 bits is what dominates a plain fp16 iteration (2e-3 relative; 5e-4 this way, against 1.7e-3 for the rounding of
//     the bf16 result); the linear terms take R and X at 22 bits.
// A and B are symmetric: only tiles on and below the diagonal are computed, and both halves written.
// All matrices of the list share each launch.
#include <type_traits>
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
constexpr int kTile = 128, kDepth = 64;        // output tile, contraction per LDS stage
constexpr int kMaxList = 24;                   // matrices per launch (they travel as kernel arguments)
constexpr int kNormParts = 256;                // partial sums of |U|^2 per matrix

struct MuonMatrix {
    const void* g;
    float* mom;
    void* w;                 // step: the weight; otherwise the output
    char* work;              // this matrix's workspace
    int r, c, m, n, mp, np;  // shape; m <= n; both rounded up to whole tiles
    int tall, splits;        // A is summed from `splits` ranges of n
    int first[3];            // first workgroup of this matrix in a product launch (A, B, X)
    float update;            // lr * s
};
struct MuonList {
    MuonMatrix a[kMaxList];
    int count, dtype, step, nesterov;
    float mu, keep, eps;     // keep = 1 - lr * decay
};

// workspace of one matrix
struct Planes { _Float16 *xh[2], *xl[2], *rh, *rl, *bh, *bl; float *da, *db, *slab; double* norm; };
__host__ __device__ inline Planes planes_of(const MuonMatrix& a) {
    Planes p;
    const int64_t x = (int64_t)a.mp * a.np, s = (int64_t)a.mp * a.mp;
    _Float16* h = (_Float16*)a.work;
    p.xh[0] = h, p.xl[0] = h + x, p.xh[1] = h + 2 * x, p.xl[1] = h + 3 * x;
    h += 4 * x;
    p.rh = h, p.rl = h + s, p.bh = h + 2 * s, p.bl = h + 3 * s;
    h += 4 * s;
    p.norm = (double*)h;
    float* f = (float*)(p.norm + kNormParts);
    p.da = f, p.db = f + a.mp, p.slab = f + 2 * a.mp;
    return p;
}

template <class T> __device__ __forceinline__ float value(const void* p, int64_t i) { return (float)((const T*)p)[i]; }
__device__ __forceinline__ float value_of(const void* p, int dtype, int64_t i) {
    return dtype == SNAG_F32 ? value<float>(p, i) : dtype == SNAG_BF16 ? value<bf16_t>(p, i) : value<f16_t>(p, i);
}

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// ---- momentum and norm: grid (kNormParts, matrices) ----------------------------------------------------------------------
__device__ __forceinline__ float update_of(const MuonList& L, float g, float m) { return L.nesterov ? fmaf(1.f - L.mu, g, L.mu * m) : m; }

template <int DT>
__global__ __launch_bounds__(256) void muon_norm_kernel(MuonList L) {
    const MuonMatrix& a = L.a[blockIdx.y];
    using T = std::conditional_t<DT == SNAG_F32, float, std::conditional_t<DT == SNAG_BF16, bf16_t, f16_t>>;
    const int64_t n = (int64_t)a.r * a.c;
    double s = 0.0;                                // the norm of gradients of any size: fp32 squares would end at 1e19
    auto one = [&](int64_t i) {
        float u = value<T>(a.g, i);
        if (L.step) {
            const float m = fmaf(L.mu, a.mom[i], (1.f - L.mu) * u);
            a.mom[i] = m;
            u = update_of(L, u, m);
        }
        return u;
    };
    // four neighbours a turn: their squares are summed in double as well
    const int64_t step = (int64_t)gridDim.x * 256 * 4;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += step) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) {
                const double u = (double)one(i + j);
                s += u * u;
            }
    }
    __shared__ double red[4];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) planes_of(a).norm[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// ---- X = U / (|U| + eps) as (hi, lo), padded with zeros: 64 x 64 blocks of X ----------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void muon_start_kernel(MuonList L) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const MuonMatrix& a = L.a[blockIdx.y];
    using T = std::conditional_t<DT == SNAG_F32, float, std::conditional_t<DT == SNAG_BF16, bf16_t, f16_t>>;
    const Planes p = planes_of(a);
    const int cols = a.np / 64, blocks = (a.mp / 64) * cols;
    if ((int)blockIdx.x >= blocks) return;         // the whole workgroup
    double s = p.norm[threadIdx.x];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]) + (double)L.eps;
    const float inv = (float)((double)kScaleX / norm);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int i0 = blk / cols * 64, j0 = blk % cols * 64;       // rows and columns of X
        if (a.tall) {
            __syncthreads();
            for (int u = wave; u < 64; u += 4) {                    // row j0 + u of U, column i0 + lane
                const int r = j0 + u, c = i0 + lane;
                float v = 0.f;
                if (r < a.r && c < a.c) {
                    const int64_t at = (int64_t)r * a.c + c;
                    v = value<T>(a.g, at);
                    if (L.step) v = update_of(L, v, a.mom[at]);
                }
                tile[u][lane] = v;
            }
            __syncthreads();
        }
        for (int u = wave; u < 64; u += 4) {
            const int r = i0 + u, c = j0 + lane;
            float v = 0.f;
            if (a.tall) {
                v = tile[lane][u];
            } else if (r < a.r && c < a.c) {
                const int64_t at = (int64_t)r * a.c + c;
                v = value<T>(a.g, at);
                if (L.step) v = update_of(L, v, a.mom[at]);
            }
            _Float16 hi, lo;
            split16(v * inv, hi, lo);
            p.xh[0][(int64_t)r * a.np + c] = hi;
            p.xl[0][(int64_t)r * a.np + c] = lo;
        }
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------
enum { kGram, kPoly, kApply };

struct TileAt { int matrix, i, j, split; };
template <int MODE>
__device__ __forceinline__ TileAt tile_at(const MuonList& L) {
    TileAt t;
    const int id = (int)xcd_order(blockIdx.x, gridDim.x);
    t.matrix = 0;
    while (t.matrix + 1 < L.count && id >= L.a[t.matrix + 1].first[MODE]) ++t.matrix;
    const MuonMatrix& a = L.a[t.matrix];
    int k = id - a.first[MODE];
    t.split = 0;
    if (MODE == kApply) {
        t.i = k % (a.mp / kTile);                  // the tiles of one column block read the same X
        t.j = k / (a.mp / kTile);
    } else {
        if (MODE == kGram) t.split = k % a.splits, k /= a.splits;
        t.i = (int)((sqrtf(8.f * k + 1.f) - 1.f) * 0.5f);
        while ((t.i + 1) * (t.i + 2) / 2 <= k) ++t.i;
        while (t.i * (t.i + 1) / 2 > k) --t.i;
        t.j = k - t.i * (t.i + 1) / 2;
    }
    return t;
}

// one 16-byte chunk per lane straight from global memory into LDS: the wave's 64 chunks land at lds, in lane order
__device__ __forceinline__ void to_lds(const void* src, void* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds((SNAG_GLOBAL void*)src, (SNAG_LDS void*)lds, 16, 0, 0);
#endif
}

// LDS stage of a K-contiguous operand: [128 rows][64] fp16, chunk c (8 values) of row r at place c ^ (r & 7): the 32 rows a fragment reads
// at once then spread over all banks.
__device__ __forceinline__ void stage_rows(const _Float16* src, int ld, int row0, int k0, _Float16* lds, int wave, int lane) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int r = (u * 4 + wave) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
        to_lds(src + (int64_t)(row0 + r) * ld + k0 + c * 8, lds + (u * 4 + wave) * 512);
    }
}
__device__ __forceinline__ f16x8 frag_rows(const _Float16* lds, int row, int kb, int lane) {
    const int r = row + (lane & 31);
    return *(const f16x8*)(lds + r * 64 + (((kb * 2 + (lane >> 5)) ^ (r & 7)) * 8));
}
// LDS stage of X as the right operand: [64 rows of the contraction][128 columns], chunk c of row r at place c ^ 4 (r & 3): the four rows a
// transposing read takes from a 16-lane group lie in different banks.
__device__ __forceinline__ void stage_cols(const _Float16* src, int ld, int k0, int col0, _Float16* lds, int wave, int lane) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int r = (u * 4 + wave) * 4 + (lane >> 4), c = (lane & 15) ^ ((r & 3) << 2);
        to_lds(src + (int64_t)(k0 + r) * ld + col0 + c * 8, lds + (u * 4 + wave) * 512);
    }
}
__device__ __forceinline__ f16x8 frag_cols(const _Float16* lds, int col, int kb, int lane) {
    union { f16x8 f; s16x4 h[2]; } v;
    const int r = kb * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2), n = col + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int row = r + 4 * w;
        const _Float16* p = lds + row * 128 + (((n >> 3) ^ ((row & 3) << 2)) * 8) + (n & 7);
#if defined(__HIP_DEVICE_COMPILE__)
        v.h[w] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)p);
#endif
    }
    return v.f;
}

// What a 32 x 32 block of the product becomes.  acc: register i of lane (h, l) = element (row0 + 8 (i / 4) + 4 h + i % 4, col0 + l).
template <int MODE>
__device__ __forceinline__ void finish(const MuonList& L, const MuonMatrix& a, const Planes& p, const f32x16& acc, int row0, int col0, bool mirror, int from, bool last, int lane) {
    const int h = lane >> 5, col = col0 + (lane & 31);
    if constexpr (MODE == kApply) {
        const _Float16 *xh = p.xh[from], *xl = p.xl[from];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int row = row0 + 8 * g + 4 * h;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t at = (int64_t)(row + j) * a.np + col;
                const float x = (float)xh[at] + (float)xl[at];                         // times 2^14
                y[j] = fmaf(kNsA + p.db[row + j], x, acc[4 * g + j] * (1.f / kScaleA));
            }
            if (!last) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t at = (int64_t)(row + j) * a.np + col;
                    _Float16 hi, lo;
                    split16(y[j], hi, lo);
                    p.xh[from ^ 1][at] = hi;
                    p.xl[from ^ 1][at] = lo;
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (row + j >= a.m || col >= a.n) continue;
                const int64_t at = a.tall ? (int64_t)col * a.c + row + j : (int64_t)(row + j) * a.c + col;
                float v = y[j] * (1.f / kScaleX);
                if (L.step) v = fmaf(-a.update, v, L.keep * value_of(a.w, L.dtype, at));
                if (L.dtype == SNAG_F32) ((float*)a.w)[at] = v;
                else if (L.dtype == SNAG_BF16) ((bf16_t*)a.w)[at] = (bf16_t)v;
                else ((f16_t*)a.w)[at] = (f16_t)v;
            }
        }
    } else {
        _Float16 *oh = MODE == kGram ? p.rh : p.bh, *ol = MODE == kGram ? p.rl : p.bl;
        float* diag = MODE == kGram ? p.da : p.db;
        const float dj = MODE == kPoly ? p.da[col] : 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int row = row0 + 8 * g + 4 * h;
            f16x4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t at = (int64_t)(row + j) * a.mp + col;
                const bool on = row + j == col;
                float v;
                if constexpr (MODE == kGram) {
                    v = acc[4 * g + j] * (1.f / (kScaleX * kScaleX));
                    if (on) diag[col] = v;
                    v *= kScaleA;
                } else {
                    const float sq = acc[4 * g + j] * (1.f / kScaleA), r = (float)p.rh[at] + (float)p.rl[at], di = p.da[row + j];      // both times 2^13
                    if (on) diag[col] = fmaf(kNsB, di, kNsC * fmaf(di, di, sq * (1.f / kScaleA)));
                    v = fmaf(fmaf(kNsC, di + dj, kNsB), r, kNsC * sq);
                }
                _Float16 vh, vl;
                split16(on ? 0.f : v, vh, vl);
                hi[j] = vh, lo[j] = vl;
                oh[at] = vh;
                ol[at] = vl;
            }
            if (mirror) {
                *(f16x4*)(oh + (int64_t)col * a.mp + row) = hi;
                *(f16x4*)(ol + (int64_t)col * a.mp + row) = lo;
            }
        }
    }
}

// 128 x 128 tile, four waves of 64 x 64; PLANES 1: hi hi, 2: hi hi + hi lo + lo hi.  Two LDS stages filled straight from memory, one ahead.
template <int MODE, int PLANES>
__global__ __launch_bounds__(256) void muon_product_kernel(MuonList L, int from, int last) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16* lds = (_Float16*)smem;
    constexpr int kOperand = kTile * kDepth, kStage = 2 * PLANES * kOperand;     // in fp16 values
    const int lane = threadIdx.x & 63, wave = wave_id_uniform();
    const TileAt t = tile_at<MODE>(L);
    const MuonMatrix& a = L.a[t.matrix];
    const Planes p = planes_of(a);
    const _Float16 *ah[2], *bh[2];
    if (MODE == kGram) ah[0] = bh[0] = p.xh[from], ah[1] = bh[1] = p.xl[from];
    else if (MODE == kPoly) ah[0] = bh[0] = p.rh, ah[1] = bh[1] = p.rl;
    else ah[0] = p.bh, ah[1] = p.bl, bh[0] = p.xh[from], bh[1] = p.xl[from];
    const int lda = MODE == kGram ? a.np : a.mp;
    int k0 = 0, k1 = MODE == kGram ? a.np : a.mp;
    if (MODE == kGram && a.splits > 1) {
        const int per = (a.np / kDepth + a.splits - 1) / a.splits * kDepth;
        k0 = t.split * per;
        k1 = min(a.np, k0 + per);
    }
    auto stage = [&](int k, int s) {
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
            _Float16* base = lds + s * kStage + q * 2 * kOperand;
            stage_rows(ah[q], lda, t.i * kTile, k, base, wave, lane);
            if (MODE == kApply) stage_cols(bh[q], a.np, k, t.j * kTile, base + kOperand, wave, lane);
            else stage_rows(bh[q], lda, t.j * kTile, k, base + kOperand, wave, lane);
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    if (k0 < k1) stage(k0, 0);
    int s = 0;
    for (int k = k0; k < k1; k += kDepth, s ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's part of stage s has landed ...
        __syncthreads();                                        // ... and everybody's; everybody is done with the other stage
        if (k + kDepth < k1) stage(k + kDepth, s ^ 1);
        const _Float16* base = lds + s * kStage;
#pragma unroll
        for (int kb = 0; kb < kDepth / 16; ++kb) {
            f16x8 fa[PLANES][2], fb[PLANES][2];
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const _Float16* o = base + q * 2 * kOperand;
                    fa[q][i] = frag_rows(o, wm + i * 32, kb, lane);
                    fb[q][i] = MODE == kApply ? frag_cols(o + kOperand, wn + i * 32, kb, lane) : frag_rows(o + kOperand, wn + i * 32, kb, lane);
                }
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[0][j], acc[i][j], 0, 0, 0);
                    if constexpr (PLANES == 2) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[1][j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[1][i], fb[0][j], acc[i][j], 0, 0, 0);
                    }
                }
#endif
        }
    }
    const int i0 = t.i * kTile + wm, j0 = t.j * kTile + wn;
    if (MODE == kGram && a.splits > 1) {
        // the range's partial tile, in register order: muon_gram_sum_kernel adds the ranges up
        const int tiles = (a.mp / kTile) * (a.mp / kTile + 1) / 2, id = t.i * (t.i + 1) / 2 + t.j;
        float* out = p.slab + ((int64_t)(t.split * tiles + id) * 16 + wave * 4) * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) *(f32x16*)(out + (i * 2 + j) * 1024) = acc[i][j];
        return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) finish<MODE>(L, a, p, acc[i][j], i0 + i * 32, j0 + j * 32, t.i != t.j, from, last != 0, lane);
}

// A from its ranges, one wave per 32 x 32 block: grid (16 x the largest number of tiles, matrices)
__global__ __launch_bounds__(64) void muon_gram_sum_kernel(MuonList L) {
    const MuonMatrix& a = L.a[blockIdx.y];
    const int tiles = (a.mp / kTile) * (a.mp / kTile + 1) / 2, id = blockIdx.x >> 4, sub = blockIdx.x & 15, lane = threadIdx.x;
    if (a.splits == 1 || id >= tiles) return;
    const Planes p = planes_of(a);
    f32x16 acc{};
    for (int s = 0; s < a.splits; ++s) acc += *(const f32x16*)(p.slab + ((int64_t)(s * tiles + id) * 16 + sub) * 1024 + lane * 16);
    int i = 0;
    while ((i + 1) * (i + 2) / 2 <= id) ++i;
    const int j = id - i * (i + 1) / 2, wave = sub >> 2, q = sub & 3;
    finish<kGram>(L, a, p, acc, i * kTile + (wave >> 1) * 64 + (q >> 1) * 32, j * kTile + (wave & 1) * 64 + (q & 1) * 32, i != j, 0, false, lane);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static int pad_tile(int n) { return (n + kTile - 1) / kTile * kTile; }

// A has few tiles when m is small, and its contraction is the long side: cut it until the launch has about one workgroup per CU, never below
// four LDS stages a range.
static int gram_splits(int mp, int np) {
    const int tiles = (mp / kTile) * (mp / kTile + 1) / 2, stages = np / kDepth;
    int s = 256 / tiles;
    if (s > stages / 4) s = stages / 4;
    return s < 1 ? 1 : s;
}

static int64_t matrix_bytes(int r, int c) {
    const int mp = pad_tile(r < c ? r : c), np = pad_tile(r < c ? c : r), s = gram_splits(mp, np);
    const int64_t x = (int64_t)mp * np, q = (int64_t)mp * mp, tiles = (int64_t)(mp / kTile) * (mp / kTile + 1) / 2;
    const int64_t n = 8 * x + 8 * q + 8 * kNormParts + 8 * (int64_t)mp + (s > 1 ? 4 * s * tiles * kTile * kTile : 0);
    return (n + 255) / 256 * 256;
}

template <int MODE>
static int product(const MuonList& L, int from, int last, hipStream_t st) {
    const MuonMatrix& e = L.a[L.count - 1];
    const int t = e.mp / kTile;
    const int n = e.first[MODE] + (MODE == kApply ? t * (e.np / kTile) : t * (t + 1) / 2 * (MODE == kGram ? e.splits : 1));
    const int planes = L.dtype == SNAG_F32 ? 2 : 1;
    const size_t lds = (size_t)2 * 2 * planes * kTile * kDepth * sizeof(_Float16);
    if (planes == 2) {
        static const hipError_t grown = hipFuncSetAttribute((const void*)muon_product_kernel<MODE, 2>, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * 2 * 2 * kTile * kDepth * 2);
        SNAG_REQUIRE(grown == hipSuccess, SNAG_ERR_LAUNCH, "muon: %s", hipGetErrorString(grown));
        muon_product_kernel<MODE, 2><<<dim3(n), 256, lds, st>>>(L, from, last);
    } else {
        muon_product_kernel<MODE, 1><<<dim3(n), 256, lds, st>>>(L, from, last);
    }
    return check_launch("muon_product");
}

// one list of at most kMaxList matrices
static int muon_go(MuonList& L, int steps, hipStream_t st) {
    int first[3] = {0, 0, 0}, blocks = 0, gram_tiles = 0;
    for (int i = 0; i < L.count; ++i) {
        MuonMatrix& a = L.a[i];
        const int t = a.mp / kTile, tri = t * (t + 1) / 2;
        for (int k = 0; k < 3; ++k) a.first[k] = first[k];
        first[kGram] += tri * a.splits;
        first[kPoly] += tri;
        first[kApply] += t * (a.np / kTile);
        const int b = (a.mp / 64) * (a.np / 64);
        blocks = b > blocks ? b : blocks;
        if (a.splits > 1 && tri > gram_tiles) gram_tiles = tri;
    }
    const dim3 gn(kNormParts, L.count), gs(blocks < 2048 ? blocks : 2048, L.count);
    switch (L.dtype) {
        case SNAG_F32: muon_norm_kernel<SNAG_F32><<<gn, 256, 0, st>>>(L); muon_start_kernel<SNAG_F32><<<gs, 256, 0, st>>>(L); break;
        case SNAG_BF16: muon_norm_kernel<SNAG_BF16><<<gn, 256, 0, st>>>(L); muon_start_kernel<SNAG_BF16><<<gs, 256, 0, st>>>(L); break;
        default: muon_norm_kernel<SNAG_F16><<<gn, 256, 0, st>>>(L); muon_start_kernel<SNAG_F16><<<gs, 256, 0, st>>>(L); break;
    }
    if (int rc = check_launch("muon_start")) return rc;
    for (int k = 0; k < steps; ++k) {
        if (int rc = product<kGram>(L, k & 1, 0, st)) return rc;
        if (gram_tiles > 0) {
            muon_gram_sum_kernel<<<dim3(16 * gram_tiles, L.count), 64, 0, st>>>(L);
            if (int rc = check_launch("muon_gram_sum")) return rc;
        }
        if (int rc = product<kPoly>(L, k & 1, 0, st)) return rc;
        if (int rc = product<kApply>(L, k & 1, k + 1 == steps, st)) return rc;
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

// All matrices of a call, kMaxList a launch; every list of launches starts at the workspace's beginning (they follow each other on the stream).
static int muon_run(const char* what, void* const* w, const void* const* g, float* const* mom, const int32_t* rows, const int32_t* cols, int count, int dtype, float lr, float mu, int nesterov,
                    float decay, int match_rms, int steps, float eps, void* work, int64_t work_bytes, void* stream) {
    if (int rc = muon_check(what, rows, cols, count, dtype)) return rc;
    SNAG_REQUIRE(steps >= 1 && steps <= 100, SNAG_ERR_ARG, "%s: %d steps", what, steps);
    SNAG_REQUIRE(eps >= 0.f, SNAG_ERR_ARG, "%s: eps %g", what, (double)eps);
    if (count == 0) return SNAG_OK;
    SNAG_REQUIRE(w != nullptr && g != nullptr, SNAG_ERR_ARG, "%s: null pointer lists", what);
    for (int i = 0; i < count; ++i) SNAG_REQUIRE(w[i] != nullptr && g[i] != nullptr && (mom == nullptr || mom[i] != nullptr), SNAG_ERR_ARG, "%s: null matrix %d", what, i);
    const int64_t need = snag_muon_work_bytes(rows, cols, count);
    SNAG_REQUIRE(work != nullptr && ((uintptr_t)work & 255) == 0 && work_bytes >= need, SNAG_ERR_ARG, "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)work_bytes,
                 (long long)need);
    for (int i0 = 0; i0 < count; i0 += kMaxList) {
        MuonList L{};
        L.count = count - i0 < kMaxList ? count - i0 : kMaxList;
        L.dtype = dtype, L.step = mom != nullptr, L.nesterov = nesterov, L.mu = mu, L.keep = 1.f - lr * decay, L.eps = eps;
        char* at = (char*)work;
        for (int i = 0; i < L.count; ++i) {
            MuonMatrix& a = L.a[i];
            const int r = rows[i0 + i], c = cols[i0 + i];
            a.g = g[i0 + i], a.w = w[i0 + i], a.mom = mom != nullptr ? mom[i0 + i] : nullptr, a.work = at;
            a.r = r, a.c = c, a.tall = r > c, a.m = r < c ? r : c, a.n = r < c ? c : r, a.mp = pad_tile(a.m), a.np = pad_tile(a.n);
            a.splits = gram_splits(a.mp, a.np);
            const double s = match_rms ? 0.2 * sqrt((double)a.n) : sqrt(r > c ? (double)r / c : 1.0);
            a.update = (float)(lr * s);
            at += matrix_bytes(r, c);
        }
        if (int rc = muon_go(L, steps, (hipStream_t)stream)) return rc;
    }
    return SNAG_OK;
}

}  // namespace snag

using namespace snag;

extern "C" SNAG_API int64_t snag_muon_work_bytes(const int32_t* rows_host, const int32_t* cols_host, int count) {
    int64_t most = 0;
    for (int i0 = 0; i0 < count && rows_host != nullptr && cols_host != nullptr; i0 += kMaxList) {
        int64_t n = 0;
        for (int i = i0; i < count && i < i0 + kMaxList; ++i)
            if (rows_host[i] >= 1 && cols_host[i] >= 1) n += matrix_bytes(rows_host[i], cols_host[i]);
        most = n > most ? n : most;
    }
    return most;
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
