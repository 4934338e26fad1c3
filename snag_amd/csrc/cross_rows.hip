// Cross attention for at most four rows (fp32: eight) per key/value head: a single new token, an entity's few modality tokens.
//
// A 32 x 32 matrix product would multiply mostly padding, and the keys and values are read once whatever is done with them: the work is
// the stream of K and V from memory, so it runs on the vector pipe.  DP / (16 bytes) lanes hold one key (16 bytes a lane), 64 / that
// many keys are worked on side by side, the R rows stay in registers; every lane group keeps a running maximum, sum and output of its
// own (fp32) and they are joined once at the end: over the groups by lane exchanges, over the waves of a problem through LDS, over the
// workgroups of a long problem by cross_combine_kernel.  The backward is one pass too: with all rows of a key/value head in one wave, d K
// and d V of a key are complete when its scores are, and only d Q is joined.
// One row, 64 x 8 heads of 128 over 4096 keys: bf16 198 us, 5.4 TB/s of keys and values, fp32 375, 5.7; three rows, 12842 x 2 heads of 64 over up to
// 24 keys in fp32: 61 us, backward 99.
#include "cross.hip.h"

namespace snag {

// all-reduce over each aligned group of N lanes (N = 4 .. 32), every lane ends with the same value
template <int N>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp_f32<0xB1>(v);                        // quad_perm: lane ^ 1
    v += dpp_f32<0x4E>(v);                        // quad_perm: lane ^ 2
    if constexpr (N >= 8) v += dpp_f32<0x141>(v); // row_half_mirror: the other quad of the eight
    if constexpr (N >= 16) v += dpp_f32<0x140>(v);// row_mirror: the other eight of the sixteen
    if constexpr (N >= 32) v += __shfl_xor(v, 16);
    return v;
}

// The same value of another lane group's, combined: all-reduce over the 64 / LPK groups, every lane ends with the same value.
__device__ __forceinline__ void swap16(float v, float& a, float& b) {       // the rows of 16 lanes 0, 0, 2, 2 and 1, 1, 3, 3
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
#else
    a = b = v;
#endif
}
__device__ __forceinline__ void swap32(float v, float& a, float& b) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
#else
    a = b = v;
#endif
}
template <int LPK>
__device__ __forceinline__ float slots_sum(float v) {
    float a, b;
    if constexpr (LPK <= 4) v += dpp_f32<0x124>(v);        // row_ror:4
    if constexpr (LPK <= 8) v += dpp_f32<0x128>(v);        // row_ror:8
    if constexpr (LPK <= 16) swap16(v, a, b), v = a + b;
    swap32(v, a, b);
    return a + b;
}
template <int LPK>
__device__ __forceinline__ float slots_max(float v) {
    float a, b;
    if constexpr (LPK <= 4) v = fmaxf(v, dpp_f32<0x124>(v));
    if constexpr (LPK <= 8) v = fmaxf(v, dpp_f32<0x128>(v));
    if constexpr (LPK <= 16) swap16(v, a, b), v = fmaxf(a, b);
    swap32(v, a, b);
    return fmaxf(a, b);
}

struct RowsItem { int b, hk, split, wave; bool live; };
// waves-per-problem W divides the workgroup's waves; ids of one problem's workgroups are neighbours
__device__ __forceinline__ RowsItem rows_item(const CrossArgs& a, int W) {
    const int wave = wave_id_uniform(), per_block = (int)(blockDim.x >> 6) / W;
    const int64_t item = (int64_t)blockIdx.x * per_block + wave / W, n = (int64_t)a.B * a.Hkv * a.splits;
    RowsItem r;
    r.live = item < n;
    const int64_t i = r.live ? item : 0;
    r.split = (int)(i % a.splits);
    const int64_t bh = i / a.splits;
    r.hk = (int)(bh % a.Hkv);
    r.b = (int)(bh / a.Hkv);
    r.wave = wave % W;
    return r;
}

__device__ __forceinline__ bool rows_key_seen(const CrossArgs& a, int b, int key, int len) {
    return key < len && (a.mask == nullptr || a.mask[(int64_t)b * a.mask_ld + key] != 0);
}

template <class T>
__device__ __forceinline__ void store_chunk(T* row, int col, int d, int vec, typename Chunk<T>::vec c) {
    if (vec && col < d) {
        *(typename Chunk<T>::vec*)(row + col) = c;
    } else {
#pragma unroll
        for (int j = 0; j < Chunk<T>::n; ++j)
            if (col + j < d) row[col + j] = c[j];
    }
}

template <class T, int DP, int R>
__global__ __launch_bounds__(R > 4 ? 512 : 1024) void cross_rows_fwd_kernel(CrossArgs a, int W) {
    constexpr int C = Chunk<T>::n, LPK = DP / C, NK = 64 / LPK, U = 4;
    extern __shared__ float join[];               // [waves][R][DP + 2]
    const int lane = threadIdx.x & 63, slot = lane / LPK, col = (lane % LPK) * C;
    const RowsItem it = rows_item(a, W);
    const int len = it.live ? cross_len(a, it.b) : 0;
    float q[R][C], acc[R][C], m[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int l = r < a.rows ? r / a.G : 0, head = it.hk * a.G + (r < a.rows ? r % a.G : 0);
        const auto c = load_chunk<T>((const T*)a.q + it.b * a.qsb + l * a.qsl + head * a.qsh, col, a.d, r < a.rows && it.live, a.vec_q);
#pragma unroll
        for (int j = 0; j < C; ++j) q[r][j] = (float)c[j], acc[r][j] = 0.f;
        m[r] = -INFINITY;
        sum[r] = 0.f;
    }
    const T* kb = (const T*)a.k + it.b * a.ksb + it.hk * a.ksh;
    const T* vb = (const T*)a.v + it.b * a.vsb + it.hk * a.vsh;
    const int k0 = it.split * a.per_split, k1 = min(len, k0 + a.per_split);
    for (int base = k0 + it.wave * NK * U; base < k1; base += W * NK * U) {
        typename Chunk<T>::vec kc[U], vc[U];
        bool seen[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + u * NK + slot;
            seen[u] = key < k1 && rows_key_seen(a, it.b, key, len);
            kc[u] = load_raw<T>(kb + (int64_t)key * a.ksl, col, a.d, seen[u], a.vec_k);
            vc[u] = load_raw<T>(vb + (int64_t)key * a.vsl, col, a.d, seen[u], a.vec_v);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) kc[u] = fix_tail<T>(kc[u], col, a.d, a.vec_k), vc[u] = fix_tail<T>(vc[u], col, a.d, a.vec_v);
        float s[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float t = 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) t = fmaf(q[r][j], (float)kc[u][j], t);
                s[u][r] = seen[u] ? group_sum<LPK>(t) * a.c2 : -INFINITY;
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mn = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, s[u][r]);
            const float ref = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m[r] - ref);
            m[r] = mn;
            sum[r] *= alpha;
#pragma unroll
            for (int j = 0; j < C; ++j) acc[r][j] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = __builtin_amdgcn_exp2f(s[u][r] - ref);
                sum[r] += p;
#pragma unroll
                for (int j = 0; j < C; ++j) acc[r][j] = fmaf(p, (float)vc[u][j], acc[r][j]);
            }
        }
    }
    // the lane groups of the wave
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float mn = slots_max<LPK>(m[r]);
        const float w = __builtin_amdgcn_exp2f(m[r] - (mn == -INFINITY ? 0.f : mn));
        m[r] = mn;
        sum[r] = slots_sum<LPK>(sum[r] * w);
#pragma unroll
        for (int j = 0; j < C; ++j) acc[r][j] = slots_sum<LPK>(acc[r][j] * w);
    }
    const int64_t n = (int64_t)a.B * a.H * a.Lq;
    // the waves of the problem (then the workgroup's only one): a thread per row and element
    if (W > 1) {
        constexpr int P = DP + 2;
        float* mine = join + wave_id_uniform() * R * P;
        if (slot == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int j = 0; j < C; ++j) mine[r * P + col + j] = acc[r][j];
                if (col == 0) mine[r * P + DP] = m[r], mine[r * P + DP + 1] = sum[r];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R * DP; i += blockDim.x) {
            const int r = i / DP, c = i % DP;
            if (r >= a.rows || c >= a.d) continue;
            float mn = -INFINITY, s = 0.f, o = 0.f;
            for (int w = 0; w < W; ++w) mn = fmaxf(mn, join[(w * R + r) * P + DP]);
            const float ref = mn == -INFINITY ? 0.f : mn;
            for (int w = 0; w < W; ++w) {
                const float f = __builtin_amdgcn_exp2f(join[(w * R + r) * P + DP] - ref);
                s = fmaf(f, join[(w * R + r) * P + DP + 1], s);
                o = fmaf(f, join[(w * R + r) * P + c], o);
            }
            const int l = r / a.G, head = it.hk * a.G + r % a.G;
            const int64_t at = ((int64_t)it.b * a.H + head) * a.Lq + l;
            if (a.splits > 1) {
                a.part[(it.split * n + at) * a.d + c] = o;
                float* ml = a.part + (int64_t)a.splits * n * a.d + (it.split * n + at) * 2;
                if (c == 0) ml[0] = mn, ml[1] = s;
            } else {
                const int64_t dense = (((int64_t)it.b * a.Lq + l) * a.H + head) * a.d + c;
                const float x = o * (s > 0.f ? 1.f / s : (s == 0.f ? 0.f : s));
                const T v = (T)x;
                ((T*)a.out)[dense] = v;
                if (a.out_lo != nullptr) ((T*)a.out_lo)[dense] = (T)(x - (float)v);
                if (c == 0) a.lse[at] = s == 0.f ? -INFINITY : mn + __builtin_amdgcn_logf(s);
            }
        }
        return;
    }
    if (!it.live || slot != 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= a.rows) break;
        const int l = r / a.G, head = it.hk * a.G + r % a.G;
        const int64_t at = ((int64_t)it.b * a.H + head) * a.Lq + l;
        if (a.splits > 1) {
            float* o = a.part + (it.split * n + at) * a.d;
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (col + j < a.d) o[col + j] = acc[r][j];
            if (col == 0) {
                float* ml = a.part + (int64_t)a.splits * n * a.d + (it.split * n + at) * 2;
                ml[0] = m[r];
                ml[1] = sum[r];
            }
            continue;
        }
        const float inv = sum[r] > 0.f ? 1.f / sum[r] : (sum[r] == 0.f ? 0.f : sum[r]);
        const int64_t dense = (((int64_t)it.b * a.Lq + l) * a.H + head) * a.d;
        typename Chunk<T>::vec c, e;
#pragma unroll
        for (int j = 0; j < C; ++j) c[j] = (T)(acc[r][j] * inv), e[j] = (T)(acc[r][j] * inv - (float)c[j]);
        store_chunk<T>((T*)a.out + dense, col, a.d, a.vec_o, c);
        if (a.out_lo != nullptr) store_chunk<T>((T*)a.out_lo + dense, col, a.d, a.vec_o, e);
        if (col == 0) a.lse[at] = sum[r] == 0.f ? -INFINITY : m[r] + __builtin_amdgcn_logf(sum[r]);
    }
}

template <class T, int DP, int R>
__global__ __launch_bounds__(512) void cross_rows_bwd_kernel(CrossArgs a, int W) {
    constexpr int C = Chunk<T>::n, LPK = DP / C, NK = 64 / LPK, U = 2;
    extern __shared__ float join[];               // [waves][R][DP]
    const int lane = threadIdx.x & 63, slot = lane / LPK, col = (lane % LPK) * C;
    const RowsItem it = rows_item(a, W);
    const int len = it.live ? cross_len(a, it.b) : 0;
    float q[R][C], g[R][C], dq[R][C], lse[R], delta[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool ok = r < a.rows && it.live;
        const int l = r < a.rows ? r / a.G : 0, head = it.hk * a.G + (r < a.rows ? r % a.G : 0);
        const int64_t dense = (((int64_t)it.b * a.Lq + l) * a.H + head) * a.d;
        const auto c = load_chunk<T>((const T*)a.q + it.b * a.qsb + l * a.qsl + head * a.qsh, col, a.d, ok, a.vec_q);
        const auto e = load_chunk<T>((const T*)a.dout + dense, col, a.d, ok, a.vec_o);
        const auto f = load_chunk<T>((const T*)a.o + dense, col, a.d, ok, a.vec_o);
        typename Chunk<T>::vec w{};
        if (a.o_lo != nullptr) w = load_chunk<T>((const T*)a.o_lo + dense, col, a.d, ok, a.vec_o);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < C; ++j) q[r][j] = (float)c[j], g[r][j] = (float)e[j], t = fmaf((float)e[j], (float)f[j] + (float)w[j], t), dq[r][j] = 0.f;
        delta[r] = group_sum<LPK>(t);
        const float s = ok ? a.lse[((int64_t)it.b * a.H + head) * a.Lq + l] : INFINITY;
        lse[r] = s == -INFINITY ? INFINITY : s;   // a row that sees no key: every p is 0
    }
    const T* kb = (const T*)a.k + it.b * a.ksb + it.hk * a.ksh;
    const T* vb = (const T*)a.v + it.b * a.vsb + it.hk * a.vsh;
    const int k0 = it.split * a.per_split, k1 = it.live ? min(a.Lk, k0 + a.per_split) : 0;
    for (int base = k0 + it.wave * NK * U; base < k1; base += W * NK * U) {
        typename Chunk<T>::vec kc[U], vc[U];
        bool seen[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + u * NK + slot;
            seen[u] = key < k1 && rows_key_seen(a, it.b, key, len);
            kc[u] = load_raw<T>(kb + (int64_t)key * a.ksl, col, a.d, seen[u], a.vec_k);
            vc[u] = load_raw<T>(vb + (int64_t)key * a.vsl, col, a.d, seen[u], a.vec_v);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) kc[u] = fix_tail<T>(kc[u], col, a.d, a.vec_k), vc[u] = fix_tail<T>(vc[u], col, a.d, a.vec_v);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + u * NK + slot;
            float dk[C], dv[C];
#pragma unroll
            for (int j = 0; j < C; ++j) dk[j] = dv[j] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float s = 0.f, dp = 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) s = fmaf(q[r][j], (float)kc[u][j], s), dp = fmaf(g[r][j], (float)vc[u][j], dp);
                s = group_sum<LPK>(s);
                dp = group_sum<LPK>(dp);
                const float p = seen[u] ? __builtin_amdgcn_exp2f(fmaf(s, a.c2, -lse[r])) : 0.f;
                const float ds = seen[u] ? p * (dp - delta[r]) * a.scale : 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    dv[j] = fmaf(p, g[r][j], dv[j]);
                    dk[j] = fmaf(ds, q[r][j], dk[j]);
                    dq[r][j] = fmaf(ds, (float)kc[u][j], dq[r][j]);
                }
            }
            if (key < k1) {
                typename Chunk<T>::vec ck, cv;
#pragma unroll
                for (int j = 0; j < C; ++j) ck[j] = (T)(seen[u] ? dk[j] : 0.f), cv[j] = (T)(seen[u] ? dv[j] : 0.f);
                const int64_t dense = (((int64_t)it.b * a.Lk + key) * a.Hkv + it.hk) * a.d;
                store_chunk<T>((T*)a.dk + dense, col, a.d, a.vec_o, ck);
                store_chunk<T>((T*)a.dv + dense, col, a.d, a.vec_o, cv);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < C; ++j) dq[r][j] = slots_sum<LPK>(dq[r][j]);
    if (W > 1) {
        float* mine = join + wave_id_uniform() * R * DP;
        if (slot == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < C; ++j) mine[r * DP + col + j] = dq[r][j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R * DP; i += blockDim.x) {
            const int r = i / DP, c = i % DP;
            if (r >= a.rows || c >= a.d) continue;
            float s = 0.f;
            for (int w = 0; w < W; ++w) s += join[w * R * DP + i];
            const int64_t dense = (((int64_t)it.b * a.Lq + r / a.G) * a.H + it.hk * a.G + r % a.G) * a.d + c;
            if (a.splits > 1) a.part[(int64_t)it.split * a.B * a.Lq * a.H * a.d + dense] = s;
            else ((T*)a.dq)[dense] = (T)s;
        }
        return;
    }
    if (!it.live || slot != 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= a.rows) break;
        const int l = r / a.G, head = it.hk * a.G + r % a.G;
        const int64_t dense = (((int64_t)it.b * a.Lq + l) * a.H + head) * a.d;
        if (a.splits > 1) {
            float* o = a.part + (int64_t)it.split * a.B * a.Lq * a.H * a.d + dense;
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (col + j < a.d) o[col + j] = dq[r][j];
        } else {
            typename Chunk<T>::vec c;
#pragma unroll
            for (int j = 0; j < C; ++j) c[j] = (T)dq[r][j];
            store_chunk<T>((T*)a.dq + dense, col, a.d, a.vec_o, c);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static int keys_per_step(int d, int dtype) {           // NK * U of the forward
    const int c = dtype == SNAG_F32 ? 4 : 8, dp = d <= 32 ? 32 : d <= 64 ? 64 : 128;
    return 64 / (dp / c) * 4;
}

// Waves a problem is given inside one workgroup: enough problems fill the chip with one wave each (4096 waves = 4 per SIMD); fewer are cut
// over the waves of a workgroup as long as each still has a step of keys.  (The backward, and more than four rows, need more registers than sixteen waves leave: at most eight.)
static int rows_waves(int64_t problems, int Lk, int step, bool at_most_8) {
    if (problems >= 4096 || Lk <= step) return 1;
    if (problems >= 1024 || Lk <= 4 * step) return 4;
    return at_most_8 || Lk <= 8 * step ? 8 : 16;
}

// Key ranges on different workgroups (joined by a second launch, about 5 us).  A workgroup's four rows x 32 keys a step are some 500 vector
// instructions, so 32 problems of 1500 keys on 32 of the 256 CUs are bound by those CUs' vector pipes (23 us with 8 waves a problem and with 16).
int cross_rows_splits(int B, int Hkv, int Lk, int d, int dtype) {
    const int64_t problems = (int64_t)B * Hkv;
    const int step = keys_per_step(d, dtype);
    if (problems == 0 || problems >= 256 || Lk <= 16 * step) return 1;
    const int64_t want = problems < 4 ? 64 : (256 + problems - 1) / problems, most = Lk / (4 * step);      // cross_combine_kernel joins up to 64
    return (int)(want < most ? want : most);
}

template <class T, int DP>
static void rows_launch(const CrossArgs& a, int W, bool bwd, hipStream_t st) {
    const int threads = W <= 4 ? 256 : 64 * W, per_block = threads / 64 / W;
    const int64_t items = (int64_t)a.B * a.Hkv * a.splits;
    const dim3 grid((unsigned)((items + per_block - 1) / per_block));
    const int R = a.rows;
#define GO(RR)                                                                                                            \
    do {                                                                                                                  \
        const size_t lds = W > 1 ? sizeof(float) * (threads / 64) * RR * (bwd ? DP : DP + 2) : 0;                         \
        if (bwd) cross_rows_bwd_kernel<T, DP, RR><<<grid, threads, lds, st>>>(a, W);                                      \
        else cross_rows_fwd_kernel<T, DP, RR><<<grid, threads, lds, st>>>(a, W);                                          \
    } while (0)
    switch (R) {
        case 1: GO(1); break;
        case 2: GO(2); break;
        case 3: GO(3); break;
        case 4: GO(4); break;
        default:                                       // fp32 only
            if constexpr (sizeof(T) == 4) {
                if (R <= 6) GO(6);
                else GO(8);
            }
    }
#undef GO
}

static int rows_go(CrossArgs a, int dtype, bool bwd, hipStream_t st) {
    const int step = keys_per_step(a.d, dtype);
    const int64_t problems = (int64_t)a.B * a.Hkv;
    const int W = rows_waves(problems * a.splits, range_of(a.Lk, a.splits), step, bwd || a.rows > 4);
    // a wave each where there are that many
    SNAG_REQUIRE(problems * a.splits < kLaunchWaves, SNAG_ERR_UNSUPPORTED, "cross attention: %lld problems, more than 2^32 threads in a launch", (long long)problems);
    a.per_split = range_of(a.Lk, a.splits);
#define GO(T) a.d <= 32 ? rows_launch<T, 32>(a, W, bwd, st) : a.d <= 64 ? rows_launch<T, 64>(a, W, bwd, st) : rows_launch<T, 128>(a, W, bwd, st)
    if (dtype == SNAG_F32) GO(float);
    else if (dtype == SNAG_BF16) GO(bf16_t);
    else GO(f16_t);
#undef GO
    return check_launch(bwd ? "cross_rows_bwd" : "cross_rows_fwd");
}

int cross_rows_fwd(const CrossArgs& a, int dtype, hipStream_t st) { return rows_go(a, dtype, false, st); }
int cross_rows_bwd(const CrossArgs& a, int dtype, hipStream_t st) { return rows_go(a, dtype, true, st); }

}  // namespace snag
