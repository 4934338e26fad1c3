// Cross attention, tiled backward (csrc/cross_tiles.hip.h has the scheme): d q, d k / d v, and the joins of split ranges.
//
// Two passes, each recomputing the scores: d q with 32 rows per wave (three products per key tile), d k / d v with 32 keys per wave (four).  One
// pass that did both would save two of the seven products and need atomics for one of the sides.  Bound by the matrix pipe.
// 2 x 16 heads of 128, 2048 rows, 8192 keys in bf16: d q 400 - 435 us by the card (0.95 - 1.03 PFLOP/s), d k / d v 620 - 690 (0.80 - 0.89); fp16, with the power of
// two that d scores carry, 448 and 658 (432 and 646 without).
#include "cross_tiles.hip.h"

namespace snag {

// d q: as the forward, 32 rows per wave; splits > 1: part[split][B, Lq, H, d], joined by cross_sum_kernel.
// With d_out in registers it also forms delta = sum_d d_out o and leaves stat[b, hk, row] = (lse, delta) to d k / d v, in the kernels' row order, each
// problem's rows padded to 64 with (+inf, 0): the p of such a row, and of one that sees no key, is 0.  (A pass of its own read d_out once
// more: 94 us of 587 at 320 problems of 2000 rows x 14 keys of 75.)
template <class T, int DP, int NW, int KT, bool DIRECT>
__global__ __launch_bounds__(NW * 64, (NW == 1 && (sizeof(T) == 4 || DP == 128)) || (sizeof(T) == 4 && DP == 128) ? 1 : 2) void cross_dq_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64;
    constexpr int NB = NW == 1 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) T lk[NB][KT * DP];
    __shared__ __attribute__((aligned(16))) T lv[NB][KT * DP];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id_uniform(), h = lane >> 5;
    const int64_t tiles = (a.rows + NW * 32 - 1) / (NW * 32);
    const Problem pr = problem_of(a, tiles);
    const int b = pr.b, hk = pr.hk;
    const int len = cross_len(a, b);
    const int row = (int)pr.tile * NW * 32 + wave * 32 + (lane & 31);
    const bool own = row < a.rows;
    const int l = own ? row_l(a, row) : 0, head = hk * a.G + (own ? row - l * a.G : 0);
    const T* kb = (const T*)a.k + b * a.ksb + hk * a.ksh;
    const T* vb = (const T*)a.v + b * a.vsb + hk * a.vsh;
    const int64_t dense = (((int64_t)b * a.Lq + l) * a.H + head) * a.d;

    const int t0 = pr.split * a.per_split / KT, t1 = min((len + KT - 1) / KT, t0 + a.per_split / KT);
    TileFetch<T, DP, KT, NT, DIRECT> fk, fv;
    bool byte = true;                                      // this lane's mask byte of the tile in flight
    uint64_t now = 0;                                      // seen keys of the tile that is worked on
    // DIRECT: rows behind the last key are read as the last key; keys that are not seen are zeros in LDS before they are used, and get -inf for a score
    auto fetch = [&](int t) {
        const int key0 = t * KT, end = (DIRECT ? len : a.Lk) - 1;
        fk.fetch([&](int i) { return kb + min(key0 + i, end) * a.ksl; }, lk[t % NB], a.d, a.vec_k, tid);
        fv.fetch([&](int i) { return vb + min(key0 + i, end) * a.vsl; }, lv[t % NB], a.d, a.vec_v, tid);
        if (!DIRECT) byte = mask_byte(a, b, key0, lane);
    };
    auto store = [&](int t) {
        if constexpr (!DIRECT) {
            now = seen_bits(byte, t * KT, len, lane);
            auto keep = [&](int i) { return (now >> i) & 1; };
            fk.store(keep, lk[t % NB], a.d, a.vec_k, tid);
            fv.store(keep, lv[t % NB], a.d, a.vec_v, tid);
        }
    };
    if (DIRECT ? t0 < t1 : t0 * KT < a.Lk) fetch(t0);
    typename M::Frag q[DP / 16], dout[DP / 16];
    own_row<T, DP>(q, (const T*)a.q + b * a.qsb + l * a.qsl + head * a.qsh, a.d, own, a.vec_q, lane);
    own_row<T, DP>(dout, (const T*)a.dout + dense, a.d, own, a.vec_o, lane);
    float lse = own ? a.lse[((int64_t)b * a.H + head) * a.Lq + l] : INFINITY, delta = 0.f;
    if (lse == -INFINITY) lse = INFINITY;
    {
        typename M::Frag o[DP / 16];
        own_row<T, DP>(o, (const T*)a.o + dense, a.d, own, a.vec_o, lane);
        float part[4] = {0.f, 0.f, 0.f, 0.f}, lo, hi;
        if (a.o_lo != nullptr) {
            typename M::Frag w[DP / 16];
            own_row<T, DP>(w, (const T*)a.o_lo + dense, a.d, own, a.vec_o, lane);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) part[j & 3] = fmaf((float)o[c][j] + (float)w[c][j], (float)dout[c][j], part[j & 3]);
        } else {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) part[j & 3] = fmaf((float)o[c][j], (float)dout[c][j], part[j & 3]);
        }
        halves((part[0] + part[1]) + (part[2] + part[3]), lo, hi);
        delta = lo + hi;
    }
    if (pr.split == 0) {
        // the last tile fills the padding too (at most the 32 rows behind its own)
        const int padded = (int)padded_rows(a.rows);
        float* st = a.stat + 2 * ((int64_t)b * a.Hkv + hk) * padded;
        const int64_t at = row, behind = at + NW * 32;
        if (h == 0 && at < padded) st[2 * at] = kIsHalf<T> ? lse - kHalfP : lse, st[2 * at + 1] = delta;
        if (h == 1 && behind < padded && pr.tile == tiles - 1) st[2 * behind] = INFINITY, st[2 * behind + 1] = 0.f;
    }
    if (t0 < t1) store(t0);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    [[maybe_unused]] float power = kHalfStart;             // fp16: ds and acc are times 2^power
    float ref = kIsHalf<T> ? lse - power : lse;
    for (int t = t0; t < t1; ++t) {
        tile_ready();
        if (DIRECT && (t + 1) * KT > len) {
            fk.pad(len - t * KT, lk[t % NB], tid);
            fv.pad(len - t * KT, lv[t % NB], tid);
            pad_ready();
        }
        if (t + 1 < t1) fetch(t + 1);
        const T *ck = lk[t % NB], *cv = lv[t % NB];
        const bool hide = (!DIRECT && a.mask != nullptr) || (t + 1) * KT > len;
        if constexpr (DIRECT) {
            if (hide) now = seen_bits(true, t * KT, len, lane);
        }
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            f32x16 s{}, dp{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                s = M::mma(M::template rows<DP>(ck, kt * 32, c * 16, lane), q[c], s);
                dp = M::mma(M::template rows<DP>(cv, kt * 32, c * 16, lane), dout[c], dp);
            }
            if (hide) hide_keys(s, (uint32_t)(now >> (32 * kt)), lane);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c2, -ref)) * (dp[i] - delta);
            if constexpr (kIsHalf<T>) {
                const int down = half_shift(largest(s));
                if (__any(down != 0)) {
                    power += (float)down;
                    ref = lse - power;
                    const float f = __builtin_amdgcn_exp2f((float)down);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] *= f;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[db][i] *= f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename M::Frag ds = pack<T>(s, u);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) acc[db] = M::mma(M::template cols<DP>(ck, kt * 32 + u * 16, db * 32, lane), ds, acc[db]);
            }
        }
        if (t + 1 < t1) store(t + 1);
    }
    if (!own) return;
    if (lse == INFINITY) {                                 // no key seen: zero, whatever d_out holds
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    }
    const float scale = kIsHalf<T> ? a.scale * __builtin_amdgcn_exp2f(-power) : a.scale;
    if (a.splits > 1) store_row<float, DP>(a.part + (int64_t)pr.split * a.B * a.Lq * a.H * a.d + dense, acc, scale, a.d, lane);
    else store_row<T, DP>((T*)a.dq + dense, acc, scale, a.d, lane);
}

// d k, d v: 32 keys per wave, row tiles of RT through LDS; splits > 1: part[2][split][B, Lk, Hkv, d] (d k, then d v)
template <class T, int DP, int NW, int RT, bool DIRECT>
__global__ __launch_bounds__(NW * 64, (NW == 1 && (sizeof(T) == 4 || DP == 128)) || (sizeof(T) == 4 && DP >= 64) ? 1 : 2) void cross_dkv_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64, KEYS = NW * 32;
    // 16-bit rows of 128: d k and d v take 128 registers, k another 32; v, the fourth operand, is read from LDS so that two waves fit a SIMD
    constexpr bool VLDS = sizeof(T) == 2 && DP == 128 && NW == 4;          // KEYS == 128
    __shared__ __attribute__((aligned(16))) T lvv[VLDS ? KEYS * DP : 16];
    constexpr int NB = NW == 1 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) T lq[NB][RT * DP];
    __shared__ __attribute__((aligned(16))) T lo[NB][RT * DP];
    __shared__ __attribute__((aligned(16))) float stat[2][2 * RT];
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
    [[maybe_unused]] float power = kHalfStart;             // fp16: ds and dk are times 2^power, p and dv times 2^kHalfP
    const int t0 = pr.split * a.per_split / RT, t1 = key0 < len ? min((a.rows + RT - 1) / RT, t0 + a.per_split / RT) : t0;
    if (t0 < t1) {
        TileFetch<T, DP, RT, NT, DIRECT> fq, fo;
        [[maybe_unused]] const float* st = a.stat + 2 * ((int64_t)b * a.Hkv + hk) * padded_rows(a.rows);
        // rows behind the last one are read as the last one and cleared in LDS, their p is 0
        auto fetch = [&](int t) {
            const int r0 = t * RT;
            fq.fetch([&](int i) {
                const int r = min(r0 + i, a.rows - 1), l = row_l(a, r);
                return (const T*)a.q + b * a.qsb + l * a.qsl + (hk * a.G + r - l * a.G) * a.qsh;
            }, lq[t % NB], a.d, a.vec_q, tid);
            fo.fetch([&](int i) {
                const int r = min(r0 + i, a.rows - 1), l = row_l(a, r);
                return (const T*)a.dout + (((int64_t)b * a.Lq + l) * a.H + hk * a.G + r - l * a.G) * a.d;
            }, lo[t % NB], a.d, a.vec_o, tid);
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
            for (int u = 0; u < 2 * RT / 64; ++u)
                if (wave == u % NW) __builtin_amdgcn_global_load_lds((SNAG_GLOBAL void*)(st + 2 * (int64_t)r0 + u * 64 + lane), (SNAG_LDS void*)(stat[t & 1] + u * 64), 4, 0, 0);
#endif
        };
        auto store = [&](int t) {
            auto keep = [&](int i) { return i < a.rows - t * RT; };
            fq.store(keep, lq[t % NB], a.d, a.vec_q, tid);
            fo.store(keep, lo[t % NB], a.d, a.vec_o, tid);
        };
        fetch(t0);
        if constexpr (VLDS) {
            TileFetch<T, DP, KEYS, NT, DIRECT> fv;
            const int end = (DIRECT ? len : a.Lk) - 1;
            fv.fetch([&](int i) { return (const T*)a.v + b * a.vsb + hk * a.vsh + min(key0 + i, end) * a.vsl; }, lvv, a.d, a.vec_v, tid);
            if constexpr (!DIRECT) {
                uint64_t bits[KEYS / 64];
#pragma unroll
                for (int u = 0; u < KEYS / 64; ++u) bits[u] = seen_bits(mask_byte(a, b, key0 + 64 * u, lane), key0 + 64 * u, len, lane);
                fv.store([&](int i) { return ((i < 64 ? bits[0] : bits[KEYS / 64 - 1]) >> (i & 63)) & 1; }, lvv, a.d, a.vec_v, tid);
            }
        }
        typename M::Frag k[DP / 16], v[VLDS ? 1 : DP / 16];
        own_row<T, DP>(k, (const T*)a.k + b * a.ksb + hk * a.ksh + key * a.ksl, a.d, seen, a.vec_k, lane);
        if constexpr (!VLDS) own_row<T, DP>(v, (const T*)a.v + b * a.vsb + hk * a.vsh + key * a.vsl, a.d, seen, a.vec_v, lane);
        store(t0);
        for (int t = t0; t < t1; ++t) {
            tile_ready();
            if (DIRECT && (t + 1) * RT > a.rows) {
                fq.pad(a.rows - t * RT, lq[t % NB], tid);
                fo.pad(a.rows - t * RT, lo[t % NB], tid);
                pad_ready();
            }
            if (t + 1 < t1) fetch(t + 1);
            const T *cq = lq[t % NB], *co = lo[t % NB];
#pragma unroll
            for (int rt = 0; rt < RT / 32; ++rt) {
                f32x16 s{}, dp{};
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    s = M::mma(M::template rows<DP>(cq, rt * 32, c * 16, lane), k[c], s);
                    if constexpr (VLDS) dp = M::mma(M::template rows<DP>(co, rt * 32, c * 16, lane), M::template rows<DP>(lvv, wave * 32, c * 16, lane), dp);
                    else dp = M::mma(M::template rows<DP>(co, rt * 32, c * 16, lane), v[c], dp);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    // (lse, delta) of four rows; fp16: lse - kHalfP.  Keys that are not seen go along: what they gather stays in their own lane and is dropped at the end
                    const f32x4 s0 = *(const f32x4*)(stat[t & 1] + 2 * (rt * 32 + g * 8 + h * 4)), s1 = *(const f32x4*)(stat[t & 1] + 2 * (rt * 32 + g * 8 + h * 4) + 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = 4 * g + j;
                        const float ls = j < 2 ? s0[2 * j] : s1[2 * j - 4], de = j < 2 ? s0[2 * j + 1] : s1[2 * j - 3];
                        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c2, -ls));
                        dp[i] = s[i] * (dp[i] - de);
                    }
                }
                if constexpr (kIsHalf<T>) {
                    const float to = __builtin_amdgcn_exp2f(power - kHalfP);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] *= to;
                    const int down = half_shift(largest(dp));
                    if (__any(down != 0)) {
                        power += (float)down;
                        const float f = __builtin_amdgcn_exp2f((float)down);
#pragma unroll
                        for (int i = 0; i < 16; ++i) dp[i] *= f;
#pragma unroll
                        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                            for (int i = 0; i < 16; ++i) dk[db][i] *= f;
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const typename M::Frag p = pack<T>(s, u), ds = pack<T>(dp, u);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        dv[db] = M::mma(M::template cols<DP>(co, rt * 32 + u * 16, db * 32, lane), p, dv[db]);
                        dk[db] = M::mma(M::template cols<DP>(cq, rt * 32 + u * 16, db * 32, lane), ds, dk[db]);
                    }
                }
            }
            if (t + 1 < t1) store(t + 1);
        }
    }
    if (!own) return;
    if (!seen) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = f32x16{};
    }
    const int64_t dense = (((int64_t)b * a.Lk + key) * a.Hkv + hk) * a.d, n = (int64_t)a.B * a.Lk * a.Hkv * a.d;
    const float k_scale = kIsHalf<T> ? a.scale * __builtin_amdgcn_exp2f(-power) : a.scale, v_scale = kIsHalf<T> ? 1.f / kHalfTop : 1.f;
    if (a.splits > 1) {
        store_row<float, DP>(a.part + pr.split * n + dense, dk, k_scale, a.d, lane);
        store_row<float, DP>(a.part + (a.splits + pr.split) * n + dense, dv, v_scale, a.d, lane);
    } else {
        store_row<T, DP>((T*)a.dk + dense, dk, k_scale, a.d, lane);
        store_row<T, DP>((T*)a.dv + dense, dv, v_scale, a.d, lane);
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
static int sum_ranges(const float* part, int64_t n, int ranges, void* out, hipStream_t st) {
    if (n == 0) return SNAG_OK;
    cross_sum_kernel<T><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st>>>(part, n, ranges, (T*)out);
    return check_launch("cross_sum");
}
int cross_sum(const float* part, int64_t n, int ranges, void* out, int dtype, hipStream_t st) {
    return dtype == SNAG_F32 ? sum_ranges<float>(part, n, ranges, out, st) : dtype == SNAG_BF16 ? sum_ranges<bf16_t>(part, n, ranges, out, st) : sum_ranges<f16_t>(part, n, ranges, out, st);
}

template <class T, int T4>
static int bwd(CrossArgs a, const CrossPlan& p, float* stat, hipStream_t st) {
    const int64_t nq = (int64_t)a.B * a.Lq * a.H, nk = (int64_t)a.B * a.Lk * a.Hkv;
    const bool whole = a.d == p.dp && a.vec_q && a.vec_k && a.vec_v && a.vec_o;
    // both launches are checked before the first one writes anything
    auto groups = [&](int64_t n, int waves, int ranges) { return (int64_t)a.B * a.Hkv * ((n + waves * 32 - 1) / (waves * 32)) * ranges; };
    const int64_t n_dq = groups(a.rows, p.nw_dq, p.s_dq), n_dkv = groups(a.Lk, p.nw_k, p.s_dkv);
    for (const int64_t waves : {n_dq * p.nw_dq, n_dkv * p.nw_k})
        SNAG_REQUIRE(waves < kLaunchWaves, SNAG_ERR_UNSUPPORTED, "cross attention backward: %lld waves, more than 2^32 threads in a launch", (long long)waves);
    a.stat = stat;
    if (nq > 0) {
        a.splits = p.s_dq;
        a.per_split = range_of(a.Lk, a.splits);
        const dim3 grid((unsigned)n_dq);
        const bool direct = p.nw_dq == 4 && whole && a.mask == nullptr;
#define CALL(DP)                                                                                  \
    if (direct) cross_dq_kernel<T, DP, 4, T4, true><<<grid, 256, 0, st>>>(a);                     \
    else if (p.nw_dq == 4) cross_dq_kernel<T, DP, 4, DP == 128 ? 32 : T4, false><<<grid, 256, 0, st>>>(a); \
    else if constexpr (sizeof(T) == 2 || DP < 128) cross_dq_kernel<T, DP, 1, 32, false><<<grid, 64, 0, st>>>(a)
        SNAG_CROSS_DP(CALL)
#undef CALL
        if (int rc = check_launch("cross_dq")) return rc;
        if (a.splits > 1)
            if (int rc = sum_ranges<T>(a.part, nq * a.d, a.splits, a.dq, st)) return rc;
    }
    if (nk > 0) {
        a.splits = p.s_dkv;
        a.per_split = range_of(a.rows, a.splits);
        const dim3 grid((unsigned)n_dkv);
        const bool direct = p.nw_k == 4 && whole && a.rows > 0;
#define CALL(DP)                                                                                  \
    if (direct) cross_dkv_kernel<T, DP, 4, DP == 128 ? 32 : T4, true><<<grid, 256, 0, st>>>(a);           \
    else if (p.nw_k == 4) cross_dkv_kernel<T, DP, 4, DP == 128 ? 32 : T4, false><<<grid, 256, 0, st>>>(a);\
    else if constexpr (sizeof(T) == 2 || DP < 128) cross_dkv_kernel<T, DP, 1, 32, false><<<grid, 64, 0, st>>>(a)
        SNAG_CROSS_DP(CALL)
#undef CALL
        if (int rc = check_launch("cross_dkv")) return rc;
        if (a.splits > 1) {
            if (int rc = sum_ranges<T>(a.part, nk * a.d, a.splits, a.dk, st)) return rc;
            if (int rc = sum_ranges<T>(a.part + a.splits * nk * a.d, nk * a.d, a.splits, a.dv, st)) return rc;
        }
    }
    return SNAG_OK;
}
int cross_tiles_bwd(const CrossArgs& a, const CrossPlan& p, float* stat, int dtype, hipStream_t st) {
    return dtype == SNAG_F32 ? bwd<float, 32>(a, p, stat, st) : dtype == SNAG_BF16 ? bwd<bf16_t, 64>(a, p, stat, st) : bwd<f16_t, 64>(a, p, stat, st);
}

}  // namespace snag
