// Cross attention on the matrix pipe: forward, d q, d k / d v, and the joins of split ranges.
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
#include <type_traits>
#include "cross.hip.h"

namespace snag {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x8 = __attribute__((ext_vector_type(8))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
#if defined(__HIP_DEVICE_COMPILE__)
#define SNAG_LDS __attribute__((address_space(3)))
#else
#define SNAG_LDS
#endif

// ---- fragments: 16 contraction elements of 32 rows / columns, 8 per lane ------------------------------------------------
template <class T> struct Mma {
    using Frag = __attribute__((ext_vector_type(8))) T;
    static constexpr int kPad = 8;            // LDS row padding in elements (16 bytes)
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (std::is_same_v<T, bf16_t>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
#else
        return c;
#endif
    }
    // A operand whose contraction index runs along the LDS row: rows row0 .. row0 + 31, elements col0 + 8 h + j
    static __device__ __forceinline__ Frag rows(const T* base, int pitch, int row0, int col0, int lane) {
        return *(const Frag*)(base + (row0 + (lane & 31)) * pitch + col0 + (lane >> 5) * 8);
    }
    // A operand whose contraction index runs over the LDS rows: columns col0 .. col0 + 31, LDS rows row0 + 8 (j / 4) + 4 h + j % 4.
    // The transposing read hands a group of 16 lanes a 4 x 16 block: lane t addresses row t / 4, columns 4 (t % 4), and receives column t.
    static __device__ __forceinline__ Frag cols(const T* base, int pitch, int row0, int col0, int lane) {
        const T* p = base + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * pitch + col0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        union { Frag f; s16x4 h[2]; } u;
#if defined(__HIP_DEVICE_COMPILE__)
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)p);
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SNAG_LDS s16x4*)(p + 8 * pitch));
#endif
        return u.f;
    }
};
template <> struct Mma<float> {
    using Frag = f32x8;
    static constexpr int kPad = 4;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
#endif
        return c;
    }
    static __device__ __forceinline__ Frag rows(const float* base, int pitch, int row0, int col0, int lane) {
        const f32x4* p = (const f32x4*)(base + (row0 + (lane & 31)) * pitch + col0 + (lane >> 5) * 8);
        const f32x4 a = p[0], b = p[1];
        return Frag{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    static __device__ __forceinline__ Frag cols(const float* base, int pitch, int row0, int col0, int lane) {
        Frag f;
        const float* p = base + (row0 + 4 * (lane >> 5)) * pitch + col0 + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = p[(8 * (j >> 2) + (j & 3)) * pitch];
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

// B operands of one row of d elements (the lane's own row), DP / 16 fragments of 8 elements
template <class T, int DP>
__device__ __forceinline__ void own_row(typename Mma<T>::Frag (&f)[DP / 16], const T* row, int d, bool valid, int vec, int lane) {
    constexpr int C = Chunk<T>::n;
#pragma unroll
    for (int kb = 0; kb < DP / 16; ++kb) {
        const int col = kb * 16 + (lane >> 5) * 8;
#pragma unroll
        for (int w = 0; w < 8 / C; ++w) {
            const auto c = load_chunk<T>(row, col + w * C, d, valid, vec);
#pragma unroll
            for (int j = 0; j < C; ++j) f[kb][w * C + j] = c[j];
        }
    }
}

// A tile of R rows x DP elements on its way from global memory to LDS: fetched into registers while the previous tile is worked on.
template <class T, int DP, int R, int NT>
struct TileFetch {
    static constexpr int C = Chunk<T>::n, kPerRow = DP / C, kAll = R * kPerRow, kN = (kAll + NT - 1) / NT;
    static_assert(kAll % NT == 0 || kN == 1, "tile does not divide among the threads");
    typename Chunk<T>::vec r[kN];
    // row(i) -> (pointer to the row's elements, valid); rows that are not valid become zeros, whatever memory holds there
    template <class RowPtr>
    __device__ __forceinline__ void fetch(RowPtr row, int d, int vec, int tid) {
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            const int e = u * NT + tid;
            bool valid;
            const T* p = row(e / kPerRow, valid);
            r[u] = load_chunk<T>(p, (e % kPerRow) * C, d, valid && (kAll % NT == 0 || e < kAll), vec);
        }
    }
    __device__ __forceinline__ void store(T* lds, int pitch, int tid) const {
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            const int e = u * NT + tid;
            if (kAll % NT == 0 || e < kAll) *(typename Chunk<T>::vec*)(lds + (e / kPerRow) * pitch + (e % kPerRow) * C) = r[u];
        }
    }
};

// Writes a transposed accumulator (rows = elements, column = the lane's row): 4 neighbouring elements per register quad.
template <class T, int DP>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DP / 32], float scale, int d, int vec4, int lane) {
    const int h = lane >> 5;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = db * 32 + g * 8 + h * 4;
            using V4 = __attribute__((ext_vector_type(4))) T;
            V4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (T)(acc[db][4 * g + j] * scale);
            if (vec4 && col + 4 <= d) {
                *(V4*)(row + col) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < d) row[col + j] = v[j];
            }
        }
}

struct Problem { int b, hk, split; int64_t tile; };
// workgroup -> (problem, split, tile): the tiles of one problem are neighbours, so that one XCD's L2 serves its keys
__device__ __forceinline__ Problem problem_of(const CrossArgs& a, int64_t tiles) {
    const int64_t id = xcd_order(blockIdx.x, gridDim.x);
    Problem p;
    p.tile = id % tiles;
    const int64_t rest = id / tiles;
    p.split = (int)(rest % a.splits);
    const int64_t bh = rest / a.splits;
    p.hk = (int)(bh % a.Hkv);
    p.b = (int)(bh / a.Hkv);
    return p;
}

// 0 / -inf per key of a tile, for keys a row does not see
__device__ __forceinline__ bool key_seen(const CrossArgs& a, int b, int key, int len) {
    return key < len && (a.mask == nullptr || a.mask[(int64_t)b * a.mask_ld + key] != 0);
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// Workgroup: NW waves x 32 rows; key tiles of KT.  splits > 1: per range part[split][B H Lq][d] = sum exp2(S - m) v (not normalised) and, behind
// all of those, [split][B H Lq][2] = (m, sum); cross_combine_kernel joins them.
template <class T, int DP, int NW, int KT>
__global__ __launch_bounds__(NW * 64) void cross_fwd_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64, P = DP + M::kPad;
    __shared__ __attribute__((aligned(16))) T lk[KT * P];
    __shared__ __attribute__((aligned(16))) T lv[KT * P];
    __shared__ __attribute__((aligned(16))) float bias[KT];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id_uniform(), h = lane >> 5;
    const int64_t tiles = (a.rows + NW * 32 - 1) / (NW * 32);
    const Problem pr = problem_of(a, tiles);
    const int b = pr.b, hk = pr.hk;
    const int len = cross_len(a, b);
    const int row = (int)pr.tile * NW * 32 + wave * 32 + (lane & 31);
    const bool own = row < a.rows;
    const int l = own ? row / a.G : 0, head = hk * a.G + (own ? row % a.G : 0);
    const T* kb = (const T*)a.k + b * a.ksb + hk * a.ksh;
    const T* vb = (const T*)a.v + b * a.vsb + hk * a.vsh;

    typename M::Frag q[DP / 16];
    own_row<T, DP>(q, (const T*)a.q + b * a.qsb + l * a.qsl + head * a.qsh, a.d, own, a.vec_q, lane);

    const int t0 = pr.split * a.per_split, t1 = min((len + KT - 1) / KT, t0 + a.per_split);
    TileFetch<T, DP, KT, NT> fk, fv;
    float fb = 0.f;
    auto fetch = [&](int t) {
        const int key0 = t * KT;
        fk.fetch([&](int i, bool& ok) { ok = key_seen(a, b, key0 + i, len); return kb + (int64_t)(key0 + i) * a.ksl; }, a.d, a.vec_k, tid);
        fv.fetch([&](int i, bool& ok) { ok = key_seen(a, b, key0 + i, len); return vb + (int64_t)(key0 + i) * a.vsl; }, a.d, a.vec_v, tid);
        if (tid < KT) fb = key_seen(a, b, key0 + tid, len) ? 0.f : -INFINITY;
    };
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    float m = -INFINITY, sum = 0.f;
    if (t0 < t1) fetch(t0);
    for (int t = t0; t < t1; ++t) {
        __syncthreads();
        fk.store(lk, P, tid);
        fv.store(lv, P, tid);
        if (tid < KT) bias[tid] = fb;
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
        f32x16 s[KT / 32];
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            s[kt] = f32x16{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s[kt] = M::mma(M::rows(lk, P, kt * 32, c * 16, lane), q[c], s[kt]);
        }
        if (a.mask != nullptr || (t + 1) * KT > len) {
#pragma unroll
            for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 bb = *(const f32x4*)(bias + kt * 32 + g * 8 + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[kt][4 * g + j] += bb[j];
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kt][i]);
        top = fmaxf(top, __shfl_xor(top, 32)) * a.c2;
        const float mn = fmaxf(m, top);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        sum *= alpha;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kt][i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], a.c2, -ref));
                sum += s[kt][i];
            }
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename M::Frag p = pack<T>(s[kt], u);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) acc[db] = M::mma(M::cols(lv, P, kt * 32 + u * 16, db * 32, lane), p, acc[db]);
            }
    }
    sum += __shfl_xor(sum, 32);
    if (!own) return;
    const int64_t at = ((int64_t)b * a.H + head) * a.Lq + l, n = (int64_t)a.B * a.H * a.Lq;
    if (a.splits > 1) {
        store_row<float, DP>(a.part + ((int64_t)pr.split * n + at) * a.d, acc, 1.f, a.d, a.d % 4 == 0, lane);
        if (h == 0) {
            float* ml = a.part + (int64_t)a.splits * n * a.d + ((int64_t)pr.split * n + at) * 2;
            ml[0] = m;
            ml[1] = sum;
        }
        return;
    }
    store_row<T, DP>((T*)a.out + (((int64_t)b * a.Lq + l) * a.H + head) * a.d, acc, sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum), a.d, a.vec_o, lane);
    if (h == 0) a.lse[at] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
}

// Joins the key ranges of the forward: one wave per row (b, head, l).
template <class T>
__global__ __launch_bounds__(256) void cross_combine_kernel(CrossArgs a) {
    const int64_t n = (int64_t)a.B * a.H * a.Lq, at = (int64_t)blockIdx.x * 4 + wave_id_uniform();
    const int lane = threadIdx.x & 63;
    if (at >= n) return;
    const float* ml = a.part + (int64_t)a.splits * n * a.d;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[(s * n + at) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f, o[2] = {0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float w = __builtin_amdgcn_exp2f(ml[(s * n + at) * 2] - ref), t = ml[(s * n + at) * 2 + 1];
        if (t == 0.f) continue;                       // a range none of whose keys is seen
        sum += w * t;
        const float* p = a.part + (s * n + at) * a.d;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < a.d) o[u] = fmaf(w, p[lane + 64 * u], o[u]);
    }
    const int64_t l = at % a.Lq, bh = at / a.Lq, head = bh % a.H, b = bh / a.H;
    T* out = (T*)a.out + ((b * a.Lq + l) * a.H + head) * a.d;
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < a.d) out[lane + 64 * u] = (T)(o[u] * inv);
    if (lane == 0) a.lse[at] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// delta[b, head, l] = sum_d dout o, one 16-lane group per row
template <class T>
__global__ __launch_bounds__(256) void cross_delta_kernel(CrossArgs a, float* __restrict__ delta) {
    constexpr int C = Chunk<T>::n;
    const int64_t n = (int64_t)a.B * a.Lq * a.H, at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int t = threadIdx.x & 15;
    float s = 0.f;
    if (at < n)
        for (int col = t * C; col < a.d; col += 16 * C) {
            const auto x = load_chunk<T>((const T*)a.o + at * a.d, col, a.d, true, a.vec_o);
            const auto y = load_chunk<T>((const T*)a.dout + at * a.d, col, a.d, true, a.vec_o);
#pragma unroll
            for (int j = 0; j < C; ++j) s = fmaf((float)x[j], (float)y[j], s);
        }
    s = sum16(s);
    if (at < n && t == 0) {
        const int64_t head = at % a.H, bl = at / a.H, l = bl % a.Lq, b = bl / a.Lq;
        delta[(b * a.H + head) * a.Lq + l] = s;
    }
}

// p of a row that sees no key is 0: its lse becomes +inf
__device__ __forceinline__ float usable_lse(float lse) { return lse == -INFINITY ? INFINITY : lse; }

// d q: as the forward, 32 rows per wave; splits > 1: part[split][B, Lq, H, d], joined by cross_sum_kernel
template <class T, int DP, int NW, int KT>
__global__ __launch_bounds__(NW * 64) void cross_dq_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64, P = DP + M::kPad;
    __shared__ __attribute__((aligned(16))) T lk[KT * P];
    __shared__ __attribute__((aligned(16))) T lv[KT * P];
    __shared__ __attribute__((aligned(16))) float bias[KT];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id_uniform(), h = lane >> 5;
    const int64_t tiles = (a.rows + NW * 32 - 1) / (NW * 32);
    const Problem pr = problem_of(a, tiles);
    const int b = pr.b, hk = pr.hk;
    const int len = cross_len(a, b);
    const int row = (int)pr.tile * NW * 32 + wave * 32 + (lane & 31);
    const bool own = row < a.rows;
    const int l = own ? row / a.G : 0, head = hk * a.G + (own ? row % a.G : 0);
    const T* kb = (const T*)a.k + b * a.ksb + hk * a.ksh;
    const T* vb = (const T*)a.v + b * a.vsb + hk * a.vsh;
    const int64_t at = ((int64_t)b * a.H + head) * a.Lq + l, dense = (((int64_t)b * a.Lq + l) * a.H + head) * a.d;

    typename M::Frag q[DP / 16], dout[DP / 16];
    own_row<T, DP>(q, (const T*)a.q + b * a.qsb + l * a.qsl + head * a.qsh, a.d, own, a.vec_q, lane);
    own_row<T, DP>(dout, (const T*)a.dout + dense, a.d, own, a.vec_o, lane);
    const float lse = own ? usable_lse(a.lse[at]) : INFINITY, delta = own ? a.delta[at] : 0.f;

    const int t0 = pr.split * a.per_split, t1 = min((len + KT - 1) / KT, t0 + a.per_split);
    TileFetch<T, DP, KT, NT> fk, fv;
    float fb = 0.f;
    auto fetch = [&](int t) {
        const int key0 = t * KT;
        fk.fetch([&](int i, bool& ok) { ok = key_seen(a, b, key0 + i, len); return kb + (int64_t)(key0 + i) * a.ksl; }, a.d, a.vec_k, tid);
        fv.fetch([&](int i, bool& ok) { ok = key_seen(a, b, key0 + i, len); return vb + (int64_t)(key0 + i) * a.vsl; }, a.d, a.vec_v, tid);
        if (tid < KT) fb = key_seen(a, b, key0 + tid, len) ? 0.f : -INFINITY;
    };
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    if (t0 < t1) fetch(t0);
    for (int t = t0; t < t1; ++t) {
        __syncthreads();
        fk.store(lk, P, tid);
        fv.store(lv, P, tid);
        if (tid < KT) bias[tid] = fb;
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
        const bool biased = a.mask != nullptr || (t + 1) * KT > len;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            f32x16 s{}, dp{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                s = M::mma(M::rows(lk, P, kt * 32, c * 16, lane), q[c], s);
                dp = M::mma(M::rows(lv, P, kt * 32, c * 16, lane), dout[c], dp);
            }
            if (biased) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 bb = *(const f32x4*)(bias + kt * 32 + g * 8 + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[4 * g + j] += bb[j];
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c2, -lse)) * (dp[i] - delta);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename M::Frag ds = pack<T>(s, u);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) acc[db] = M::mma(M::cols(lk, P, kt * 32 + u * 16, db * 32, lane), ds, acc[db]);
            }
        }
    }
    if (!own) return;
    if (a.splits > 1) store_row<float, DP>(a.part + (int64_t)pr.split * a.B * a.Lq * a.H * a.d + dense, acc, a.scale, a.d, a.d % 4 == 0, lane);
    else store_row<T, DP>((T*)a.dq + dense, acc, a.scale, a.d, a.vec_o, lane);
}

// d k, d v: 32 keys per wave, row tiles of 32 through LDS; splits > 1: part[2][split][B, Lk, Hkv, d] (d k, then d v)
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void cross_dkv_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64, P = DP + M::kPad, RT = 32;
    __shared__ __attribute__((aligned(16))) T lq[RT * P];
    __shared__ __attribute__((aligned(16))) T lo[RT * P];
    __shared__ __attribute__((aligned(16))) float stat[2][RT];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id_uniform(), h = lane >> 5;
    const int64_t tiles = (a.Lk + NW * 32 - 1) / (NW * 32);
    const Problem pr = problem_of(a, tiles);
    const int b = pr.b, hk = pr.hk;
    const int len = cross_len(a, b);
    const int key0 = (int)pr.tile * NW * 32, key = key0 + wave * 32 + (lane & 31);
    const bool own = key < a.Lk, seen = own && key_seen(a, b, key, len);

    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = f32x16{};
    if (key0 < len) {
        typename M::Frag k[DP / 16], v[DP / 16];
        own_row<T, DP>(k, (const T*)a.k + b * a.ksb + hk * a.ksh + (int64_t)key * a.ksl, a.d, seen, a.vec_k, lane);
        own_row<T, DP>(v, (const T*)a.v + b * a.vsb + hk * a.vsh + (int64_t)key * a.vsl, a.d, seen, a.vec_v, lane);
        const int t0 = pr.split * a.per_split, t1 = min((a.rows + RT - 1) / RT, t0 + a.per_split);
        TileFetch<T, DP, RT, NT> fq, fo;
        float fs0 = 0.f, fs1 = 0.f;
        auto fetch = [&](int t) {
            const int r0 = t * RT;
            fq.fetch([&](int i, bool& ok) {
                const int r = r0 + i, l = r / a.G, head = hk * a.G + r % a.G;
                ok = r < a.rows;
                return (const T*)a.q + b * a.qsb + l * a.qsl + head * a.qsh;
            }, a.d, a.vec_q, tid);
            fo.fetch([&](int i, bool& ok) {
                const int r = r0 + i, l = r / a.G, head = hk * a.G + r % a.G;
                ok = r < a.rows;
                return (const T*)a.dout + (((int64_t)b * a.Lq + l) * a.H + head) * a.d;
            }, a.d, a.vec_o, tid);
            if (tid < RT) {
                const int r = r0 + tid, l = r / a.G, head = hk * a.G + r % a.G;
                const int64_t at = ((int64_t)b * a.H + head) * a.Lq + l;
                fs0 = r < a.rows ? usable_lse(a.lse[at]) : INFINITY;
                fs1 = r < a.rows ? a.delta[at] : 0.f;
            }
        };
        if (t0 < t1) fetch(t0);
        for (int t = t0; t < t1; ++t) {
            __syncthreads();
            fq.store(lq, P, tid);
            fo.store(lo, P, tid);
            if (tid < RT) stat[0][tid] = fs0, stat[1][tid] = fs1;
            __syncthreads();
            if (t + 1 < t1) fetch(t + 1);
            f32x16 s{}, dp{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                s = M::mma(M::rows(lq, P, 0, c * 16, lane), k[c], s);
                dp = M::mma(M::rows(lo, P, 0, c * 16, lane), v[c], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 ls = *(const f32x4*)(&stat[0][g * 8 + h * 4]), de = *(const f32x4*)(&stat[1][g * 8 + h * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = 4 * g + j;
                    s[i] = seen ? __builtin_amdgcn_exp2f(fmaf(s[i], a.c2, -ls[j])) : 0.f;
                    dp[i] = seen ? s[i] * (dp[i] - de[j]) : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename M::Frag p = pack<T>(s, u), ds = pack<T>(dp, u);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    dv[db] = M::mma(M::cols(lo, P, u * 16, db * 32, lane), p, dv[db]);
                    dk[db] = M::mma(M::cols(lq, P, u * 16, db * 32, lane), ds, dk[db]);
                }
            }
        }
    }
    if (!own) return;
    const int64_t dense = (((int64_t)b * a.Lk + key) * a.Hkv + hk) * a.d, n = (int64_t)a.B * a.Lk * a.Hkv * a.d;
    if (a.splits > 1) {
        store_row<float, DP>(a.part + pr.split * n + dense, dk, a.scale, a.d, a.d % 4 == 0, lane);
        store_row<float, DP>(a.part + (a.splits + pr.split) * n + dense, dv, 1.f, a.d, a.d % 4 == 0, lane);
    } else {
        store_row<T, DP>((T*)a.dk + dense, dk, a.scale, a.d, a.vec_o, lane);
        store_row<T, DP>((T*)a.dv + dense, dv, 1.f, a.d, a.vec_o, lane);
    }
}

// out[i] = sum over ranges of part[range][i], in order
template <class T>
__global__ __launch_bounds__(256) void cross_sum_kernel(const float* __restrict__ part, int64_t n, int ranges, T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int r = 0; r < ranges; ++r) s += part[r * n + i];
    out[i] = (T)s;
}

// ---- host ---------------------------------------------------------------------------------------------------------------
template <class T>
static int cross_sum(const float* part, int64_t n, int ranges, void* out, hipStream_t st) {
    if (n == 0) return SNAG_OK;
    cross_sum_kernel<T><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st>>>(part, n, ranges, (T*)out);
    return check_launch("cross_sum");
}

// How many ranges a loop of `tiles` tiles is cut into when `groups` workgroups exist without cutting: enough to give each of the 256 CUs two
// workgroups, never fewer than four tiles a range (a range costs its partial result's write and read).
static int ranges_for(int64_t groups, int tiles) {
    if (groups <= 0 || groups >= 512 || tiles < 8) return 1;
    const int64_t want = (512 + groups - 1) / groups;
    return (int)(want < tiles / 4 ? want : tiles / 4);
}

struct CrossPlan { int rows_path, nw_q, nw_k, kt, dp, s_fwd, s_dq, s_dkv; };

static int elem_size(int dtype) { return dtype == SNAG_F32 ? 4 : 2; }

// rows_path: a few rows per key/value head (csrc/cross_rows.hip) -- a 32-row product would multiply mostly padding
static CrossPlan cross_plan(int dtype, int B, int Lq, int Lk, int H, int Hkv, int d) {
    CrossPlan p{};
    const int64_t rows = (int64_t)Lq * (H / Hkv), bh = (int64_t)B * Hkv;
    p.dp = d <= 32 ? 32 : d <= 64 ? 64 : 128;
    p.rows_path = rows <= 4;
    if (p.rows_path) {
        p.s_fwd = p.s_dq = cross_rows_splits(B, Hkv, Lk, d, dtype);
        p.s_dkv = 1;
        return p;
    }
    p.nw_q = rows > 32 ? 4 : 1;
    p.nw_k = Lk > 32 ? 4 : 1;
    p.kt = dtype == SNAG_F32 || p.nw_q == 1 ? 32 : 64;
    p.s_fwd = p.s_dq = ranges_for(bh * ((rows + p.nw_q * 32 - 1) / (p.nw_q * 32)), (Lk + p.kt - 1) / p.kt);
    p.s_dkv = ranges_for(bh * ((Lk + p.nw_k * 32 - 1) / (p.nw_k * 32)), (int)((rows + 31) / 32));
    return p;
}

static int64_t fwd_part_floats(const CrossPlan& p, int64_t n, int d) { return p.s_fwd > 1 ? p.s_fwd * n * (d + 2) : 0; }
static int64_t bwd_part_floats(const CrossPlan& p, int64_t nq, int64_t nk, int d) {
    const int64_t dq = p.s_dq > 1 ? p.s_dq * nq * d : 0, dkv = p.s_dkv > 1 ? 2 * p.s_dkv * nk * d : 0;
    return dq > dkv ? dq : dkv;
}

#define SNAG_CROSS_DP(CALL)                  \
    switch (p.dp) {                          \
        case 32: CALL(32); break;            \
        case 64: CALL(64); break;            \
        default: CALL(128); break;           \
    }

template <class T, int KT4>
static int launch_fwd(const CrossArgs& a, const CrossPlan& p, hipStream_t st) {
    const int64_t tiles = (a.rows + p.nw_q * 32 - 1) / (p.nw_q * 32), n = (int64_t)a.B * a.Hkv * tiles * a.splits;
    SNAG_REQUIRE(n < (int64_t)1 << 31, SNAG_ERR_UNSUPPORTED, "cross attention: %lld workgroups", (long long)n);
    const dim3 grid((unsigned)n);
#define CALL(DP) if (p.nw_q == 4) cross_fwd_kernel<T, DP, 4, KT4><<<grid, 256, 0, st>>>(a); else cross_fwd_kernel<T, DP, 1, 32><<<grid, 64, 0, st>>>(a)
    SNAG_CROSS_DP(CALL)
#undef CALL
    return check_launch("cross_fwd");
}

template <class T>
static int combine(const CrossArgs& a, hipStream_t st) {
    const int64_t n = (int64_t)a.B * a.H * a.Lq;
    cross_combine_kernel<T><<<dim3((unsigned)((n + 3) / 4)), 256, 0, st>>>(a);
    return check_launch("cross_combine");
}

template <class T, int KT4>
static int launch_bwd(CrossArgs a, const CrossPlan& p, float* delta, hipStream_t st) {
    const int64_t nq = (int64_t)a.B * a.Lq * a.H, nk = (int64_t)a.B * a.Lk * a.Hkv;
    a.delta = delta;
    if (nq > 0) {
        cross_delta_kernel<T><<<dim3((unsigned)((nq + 15) / 16)), 256, 0, st>>>(a, delta);
        if (int rc = check_launch("cross_delta")) return rc;
        a.splits = p.s_dq;
        a.per_split = (int)(((a.Lk + p.kt - 1) / p.kt + a.splits - 1) / a.splits);
        const int64_t tiles = (a.rows + p.nw_q * 32 - 1) / (p.nw_q * 32), n = (int64_t)a.B * a.Hkv * tiles * a.splits;
        SNAG_REQUIRE(n < (int64_t)1 << 31, SNAG_ERR_UNSUPPORTED, "cross attention: %lld workgroups", (long long)n);
        const dim3 grid((unsigned)n);
#define CALL(DP) if (p.nw_q == 4) cross_dq_kernel<T, DP, 4, KT4><<<grid, 256, 0, st>>>(a); else cross_dq_kernel<T, DP, 1, 32><<<grid, 64, 0, st>>>(a)
        SNAG_CROSS_DP(CALL)
#undef CALL
        if (int rc = check_launch("cross_dq")) return rc;
        if (a.splits > 1)
            if (int rc = cross_sum<T>(a.part, nq * a.d, a.splits, a.dq, st)) return rc;
    }
    if (nk > 0) {
        a.splits = p.s_dkv;
        a.per_split = (a.rows + 31) / 32 > 0 ? ((a.rows + 31) / 32 + a.splits - 1) / a.splits : 1;
        const int64_t tiles = (a.Lk + p.nw_k * 32 - 1) / (p.nw_k * 32), n = (int64_t)a.B * a.Hkv * tiles * a.splits;
        SNAG_REQUIRE(n < (int64_t)1 << 31, SNAG_ERR_UNSUPPORTED, "cross attention: %lld workgroups", (long long)n);
        const dim3 grid((unsigned)n);
#define CALL(DP) if (p.nw_k == 4) cross_dkv_kernel<T, DP, 4><<<grid, 256, 0, st>>>(a); else cross_dkv_kernel<T, DP, 1><<<grid, 64, 0, st>>>(a)
        SNAG_CROSS_DP(CALL)
#undef CALL
        if (int rc = check_launch("cross_dkv")) return rc;
        if (a.splits > 1) {
            if (int rc = cross_sum<T>(a.part, nk * a.d, a.splits, a.dk, st)) return rc;
            if (int rc = cross_sum<T>(a.part + a.splits * nk * a.d, nk * a.d, a.splits, a.dv, st)) return rc;
        }
    }
    return SNAG_OK;
}

static int cross_shapes(int dtype, int B, int Lq, int Lk, int H, int Hkv, int d) {
    SNAG_REQUIRE(dtype == SNAG_F32 || dtype == SNAG_BF16 || dtype == SNAG_F16, SNAG_ERR_ARG, "cross attention: dtype %d", dtype);
    SNAG_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && H >= 1 && Hkv >= 1, SNAG_ERR_ARG, "cross attention: negative or empty size (B %d, Lq %d, Lk %d, H %d, Hkv %d)", B, Lq, Lk, H, Hkv);
    SNAG_REQUIRE(H % Hkv == 0, SNAG_ERR_ARG, "cross attention: %d heads are not a multiple of %d key/value heads", H, Hkv);
    SNAG_REQUIRE(d >= 1 && d <= SNAG_CROSS_MAX_HEAD_DIM, SNAG_ERR_UNSUPPORTED, "cross attention: head dimension %d is not in 1..%d", d, SNAG_CROSS_MAX_HEAD_DIM);
    SNAG_REQUIRE((int64_t)Lq * (H / Hkv) <= (1 << 30) && (int64_t)Lk <= (1 << 30), SNAG_ERR_UNSUPPORTED, "cross attention: more than 2^30 rows or keys in one problem");
    return SNAG_OK;
}

// the part of the arguments that the two directions share; strides_host = {q batch, position, head, k ..., v ...}
static int cross_args(CrossArgs& a, const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int d, const int64_t* s,
                      const void* lens, int lens_bytes, const uint8_t* mask, int64_t mask_ld, float scale) {
    if (int rc = cross_shapes(dtype, B, Lq, Lk, H, Hkv, d)) return rc;
    SNAG_REQUIRE(s != nullptr, SNAG_ERR_ARG, "cross attention: null strides");
    const bool hasq = B > 0 && Lq > 0, hask = B > 0 && Lk > 0;
    SNAG_REQUIRE(!hasq || q != nullptr, SNAG_ERR_ARG, "cross attention: null q");
    SNAG_REQUIRE(!hask || (k != nullptr && v != nullptr), SNAG_ERR_ARG, "cross attention: null k / v");
    SNAG_REQUIRE(lens == nullptr || lens_bytes == 4 || lens_bytes == 8, SNAG_ERR_ARG, "cross attention: lens_bytes %d", lens_bytes);
    SNAG_REQUIRE(mask == nullptr || mask_ld >= 0, SNAG_ERR_ARG, "cross attention: mask pitch %lld", (long long)mask_ld);
    SNAG_REQUIRE(scale > 0.f && scale < INFINITY, SNAG_ERR_ARG, "cross attention: scale %g is not positive and finite", (double)scale);
    a.q = q, a.k = k, a.v = v;
    a.qsb = s[0], a.qsl = s[1], a.qsh = s[2], a.ksb = s[3], a.ksl = s[4], a.ksh = s[5], a.vsb = s[6], a.vsl = s[7], a.vsh = s[8];
    a.B = B, a.Lq = Lq, a.Lk = Lk, a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.d = d, a.rows = Lq * a.G;
    a.lens = lens, a.lens_bytes = lens_bytes, a.mask = mask, a.mask_ld = mask_ld;
    a.scale = scale, a.c2 = scale * 1.44269504088896340736f;
    const int c = 16 / elem_size(dtype);
    auto vec = [&](const void* p, const int64_t* t) { return d % c == 0 && aligned16(p) && t[0] % c == 0 && t[1] % c == 0 && t[2] % c == 0; };
    a.vec_q = vec(q, s), a.vec_k = vec(k, s + 3), a.vec_v = vec(v, s + 6);
    return SNAG_OK;
}

}  // namespace snag

using namespace snag;

extern "C" SNAG_API int64_t snag_cross_work_floats(int dtype, int B, int Lq, int Lk, int H, int Hkv, int d, int backward) {
    if (cross_shapes(dtype, B, Lq, Lk, H, Hkv, d) != SNAG_OK || B == 0) return 0;
    const CrossPlan p = cross_plan(dtype, B, Lq, Lk, H, Hkv, d);
    const int64_t nq = (int64_t)B * Lq * H, nk = (int64_t)B * Lk * Hkv;
    return backward ? (nq + 3) / 4 * 4 + bwd_part_floats(p, nq, nk, d) : fwd_part_floats(p, nq, d);
}

extern "C" SNAG_API int snag_cross_fwd(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int d,
                                       const int64_t* strides_host, const void* kv_lens, int lens_bytes, const uint8_t* key_mask, int64_t mask_ld, float scale,
                                       void* out, float* lse, float* work, int64_t work_floats, void* stream) {
    CrossArgs a{};
    if (int rc = cross_args(a, q, k, v, dtype, B, Lq, Lk, H, Hkv, d, strides_host, kv_lens, lens_bytes, key_mask, mask_ld, scale)) return rc;
    if (B == 0 || Lq == 0) return SNAG_OK;
    SNAG_REQUIRE(out != nullptr && lse != nullptr, SNAG_ERR_ARG, "cross attention: null out / lse");
    const CrossPlan p = cross_plan(dtype, B, Lq, Lk, H, Hkv, d);
    const int64_t need = snag_cross_work_floats(dtype, B, Lq, Lk, H, Hkv, d, 0);
    SNAG_REQUIRE(need == 0 || (work != nullptr && work_floats >= need), SNAG_ERR_ARG, "cross attention: workspace of %lld floats, %lld needed", (long long)work_floats, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    a.out = out, a.lse = lse, a.part = work, a.splits = p.s_fwd;
    a.vec_o = d % (16 / elem_size(dtype)) == 0 && aligned16(out);
    int rc;
    if (p.rows_path) {
        rc = cross_rows_fwd(a, dtype, st);
    } else {
        a.per_split = ((Lk + p.kt - 1) / p.kt + a.splits - 1) / a.splits;
        rc = dtype == SNAG_F32 ? launch_fwd<float, 32>(a, p, st) : dtype == SNAG_BF16 ? launch_fwd<bf16_t, 64>(a, p, st) : launch_fwd<f16_t, 64>(a, p, st);
    }
    if (rc != SNAG_OK || a.splits == 1) return rc;
    return dtype == SNAG_F32 ? combine<float>(a, st) : dtype == SNAG_BF16 ? combine<bf16_t>(a, st) : combine<f16_t>(a, st);
}

extern "C" SNAG_API int snag_cross_bwd(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int d,
                                       const int64_t* strides_host, const void* kv_lens, int lens_bytes, const uint8_t* key_mask, int64_t mask_ld, float scale,
                                       const void* out, const float* lse, const void* d_out, void* d_q, void* d_k, void* d_v,
                                       float* work, int64_t work_floats, void* stream) {
    CrossArgs a{};
    if (int rc = cross_args(a, q, k, v, dtype, B, Lq, Lk, H, Hkv, d, strides_host, kv_lens, lens_bytes, key_mask, mask_ld, scale)) return rc;
    if (B == 0 || (Lq == 0 && Lk == 0)) return SNAG_OK;
    SNAG_REQUIRE(Lq == 0 || (out != nullptr && lse != nullptr && d_out != nullptr && d_q != nullptr), SNAG_ERR_ARG, "cross attention backward: null out / lse / d_out / d_q");
    SNAG_REQUIRE(Lk == 0 || (d_k != nullptr && d_v != nullptr), SNAG_ERR_ARG, "cross attention backward: null d_k / d_v");
    const CrossPlan p = cross_plan(dtype, B, Lq, Lk, H, Hkv, d);
    const int64_t need = snag_cross_work_floats(dtype, B, Lq, Lk, H, Hkv, d, 1);
    SNAG_REQUIRE(need == 0 || (work != nullptr && work_floats >= need), SNAG_ERR_ARG, "cross attention backward: workspace of %lld floats, %lld needed", (long long)work_floats, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    a.o = out, a.lse = (float*)lse, a.dout = d_out, a.dq = d_q, a.dk = d_k, a.dv = d_v;
    a.vec_o = d % (16 / elem_size(dtype)) == 0 && aligned16(out) && aligned16(d_out) && aligned16(d_q) && aligned16(d_k) && aligned16(d_v);
    a.part = work + ((int64_t)B * Lq * H + 3) / 4 * 4;
    if (p.rows_path && Lq > 0) {
        a.splits = p.s_dq;
        if (int rc = cross_rows_bwd(a, dtype, st)) return rc;
        if (a.splits == 1) return SNAG_OK;
        const int64_t n = (int64_t)B * Lq * H * d;
        return dtype == SNAG_F32 ? cross_sum<float>(a.part, n, a.splits, d_q, st) : dtype == SNAG_BF16 ? cross_sum<bf16_t>(a.part, n, a.splits, d_q, st) : cross_sum<f16_t>(a.part, n, a.splits, d_q, st);
    }
    CrossPlan pb = p;
    if (p.rows_path) pb.nw_q = 1, pb.nw_k = 4, pb.kt = 32, pb.s_dq = pb.s_dkv = 1;      // no rows: d k = d v = 0
    return dtype == SNAG_F32 ? launch_bwd<float, 32>(a, pb, work, st) : dtype == SNAG_BF16 ? launch_bwd<bf16_t, 64>(a, pb, work, st) : launch_bwd<f16_t, 64>(a, pb, work, st);
}
