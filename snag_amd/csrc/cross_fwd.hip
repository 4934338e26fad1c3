// Cross attention, tiled forward (csrc/cross_tiles.hip.h has the scheme) and the join of key ranges.
//
// Bound by the matrix pipe and, nearly as much, by the vector pipe's exponentials: 64 keys x 32 rows of 128 elements are 1024 cycles of products and
// about 900 of softmax per wave, which two waves per SIMD overlap (hence at most 256 registers).  The running maximum is only moved -- and the
// 64 accumulators rescaled -- when a score passes it by more than 8 (in log2): until then p stays below 2^8, which costs nothing in fp32 sums or
// in the 8 / 11 significant bits of the rounded p.
// 2 x 16 heads of 128, 2048 rows, 8192 keys in bf16: 300 - 340 us by the card, 0.81 - 0.92 PFLOP/s (a 4096^3 library product: 1.24); 4 x 16 x 1024 x 2048
// in fp32: 672 us, 102 TFLOP/s (library: 134 - 154).
#include "cross_tiles.hip.h"

namespace snag {

constexpr float kSlack = 8.f;

// Workgroup: NW waves x 32 rows; key tiles of KT.  splits > 1: per range part[split][B H Lq][d] = sum exp2(S - m) v (not normalised) and, behind
// all of those, [split][B H Lq][2] = (m, sum); cross_combine_kernel joins them.
template <class T, int DP, int NW, int KT, bool DIRECT>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 4 && (NW == 1 || DP == 128) ? 1 : 2) void cross_fwd_kernel(CrossArgs a) {
    using M = Mma<T>;
    constexpr int NT = NW * 64;
    constexpr int NB = NW == 1 ? 1 : 2;                    // one wave holds its next tile in registers until it is done with this one
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
    typename M::Frag q[DP / 16];
    own_row<T, DP>(q, (const T*)a.q + b * a.qsb + l * a.qsl + head * a.qsh, a.d, own, a.vec_q, lane);
    if (t0 < t1) store(t0);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
    float m = -INFINITY, sum = 0.f;                        // m: what the exponentials are relative to, within kSlack of the maximum
    for (int t = t0; t < t1; ++t) {
        tile_ready();
        if (DIRECT && (t + 1) * KT > len) {
            fk.pad(len - t * KT, lk[t % NB], tid);
            fv.pad(len - t * KT, lv[t % NB], tid);
            pad_ready();
        }
        if (t + 1 < t1) fetch(t + 1);
        const T *ck = lk[t % NB], *cv = lv[t % NB];
        f32x16 s[KT / 32];
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt) {
            s[kt] = f32x16{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) s[kt] = M::mma(M::template rows<DP>(ck, kt * 32, c * 16, lane), q[c], s[kt]);
        }
        if ((!DIRECT && a.mask != nullptr) || (t + 1) * KT > len) {
            if constexpr (DIRECT) now = seen_bits(true, t * KT, len, lane);
#pragma unroll
            for (int kt = 0; kt < KT / 32; ++kt) hide_keys(s[kt], (uint32_t)(now >> (32 * kt)), lane);
        }
        float top = -INFINITY, lo, hi;
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kt][i]);
        halves(top, lo, hi);
        top = fmaxf(lo, hi) * a.c2;
        if (__any(top > m + kSlack)) {                     // also the first score a row sees: m is -inf until then
            const float mn = fmaxf(m, top), alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= alpha;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kt][i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], a.c2, -ref));
                part[i & 3] += s[kt][i];
            }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int kt = 0; kt < KT / 32; ++kt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename M::Frag p = pack<T>(s[kt], u);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) acc[db] = M::mma(M::template cols<DP>(cv, kt * 32 + u * 16, db * 32, lane), p, acc[db]);
            }
        if (t + 1 < t1) store(t + 1);
    }
    float lo, hi;
    halves(sum, lo, hi);
    sum = lo + hi;
    if (!own) return;
    const int64_t at = ((int64_t)b * a.H + head) * a.Lq + l, n = (int64_t)a.B * a.H * a.Lq;
    if (a.splits > 1) {
        store_row<float, DP>(a.part + ((int64_t)pr.split * n + at) * a.d, acc, 1.f, a.d, lane);
        if (h == 0) {
            float* ml = a.part + (int64_t)a.splits * n * a.d + ((int64_t)pr.split * n + at) * 2;
            ml[0] = m;
            ml[1] = sum;
        }
        return;
    }
    const int64_t dense = (((int64_t)b * a.Lq + l) * a.H + head) * a.d;
    store_row<T, DP>((T*)a.out + dense, acc, sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum), a.d, lane, a.out_lo != nullptr ? (T*)a.out_lo + dense : nullptr);
    if (h == 0) a.lse[at] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
}

// Joins the key ranges of the forward (at most 64): one wave per row (b, head, l), lane s looks at range s.
template <class T>
__global__ __launch_bounds__(256) void cross_combine_kernel(CrossArgs a) {
    const int64_t n = (int64_t)a.B * a.H * a.Lq, at = (int64_t)blockIdx.x * 4 + wave_id_uniform();
    const int lane = threadIdx.x & 63;
    if (at >= n) return;
    const float* ml = a.part + (int64_t)a.splits * n * a.d;
    const bool mine = lane < a.splits;
    const float ms = mine ? ml[(lane * n + at) * 2] : -INFINITY, ts = mine ? ml[(lane * n + at) * 2 + 1] : 0.f;
    const float m = max64(ms), ref = m == -INFINITY ? 0.f : m;
    const float w = ts == 0.f ? 0.f : __builtin_amdgcn_exp2f(ms - ref);       // 0: a range none of whose keys is seen
    const float sum = sum64(w * ts);
    float o[2] = {0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s));
        const float* p = a.part + (s * n + at) * a.d;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float x = lane + 64 * u < a.d ? p[lane + 64 * u] : 0.f;
            o[u] = f == 0.f ? o[u] : fmaf(f, x, o[u]);
        }
    }
    const int64_t l = at % a.Lq, bh = at / a.Lq, head = bh % a.H, b = bh / a.H;
    const int64_t dense = ((b * a.Lq + l) * a.H + head) * a.d;
    T* out = (T*)a.out + dense;
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < a.d) {
            const T v = (T)(o[u] * inv);
            out[lane + 64 * u] = v;
            if (a.out_lo != nullptr) ((T*)a.out_lo)[dense + lane + 64 * u] = (T)(o[u] * inv - (float)v);
        }
    if (lane == 0) a.lse[at] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
template <class T, int KT4>
static void go(const CrossArgs& a, const CrossPlan& p, dim3 grid, hipStream_t st) {
    const bool direct = p.nw_fwd == 4 && a.mask == nullptr && a.d == p.dp && a.vec_k && a.vec_v;
#define CALL(DP)                                                                                   \
    if (direct) cross_fwd_kernel<T, DP, 4, KT4, true><<<grid, 256, 0, st>>>(a);                    \
    else if (p.nw_fwd == 4) cross_fwd_kernel<T, DP, 4, KT4, false><<<grid, 256, 0, st>>>(a);         \
    else cross_fwd_kernel<T, DP, 1, 32, false><<<grid, 64, 0, st>>>(a)
    SNAG_CROSS_DP(CALL)
#undef CALL
}

int cross_tiles_fwd(const CrossArgs& a, const CrossPlan& p, int dtype, hipStream_t st) {
    const int64_t tiles = (a.rows + p.nw_fwd * 32 - 1) / (p.nw_fwd * 32), n = (int64_t)a.B * a.Hkv * tiles * a.splits;
    SNAG_REQUIRE(n * p.nw_fwd < kLaunchWaves, SNAG_ERR_UNSUPPORTED, "cross attention: %lld workgroups, more than 2^32 threads in a launch", (long long)n);
    const dim3 grid((unsigned)n);
    if (dtype == SNAG_F32) go<float, 32>(a, p, grid, st);
    else if (dtype == SNAG_BF16) go<bf16_t, 64>(a, p, grid, st);
    else go<f16_t, 64>(a, p, grid, st);
    return check_launch("cross_fwd");
}

int cross_combine(const CrossArgs& a, int dtype, hipStream_t st) {
    const int64_t n = (int64_t)a.B * a.H * a.Lq;
    const dim3 grid((unsigned)((n + 3) / 4));
    if (dtype == SNAG_F32) cross_combine_kernel<float><<<grid, 256, 0, st>>>(a);
    else if (dtype == SNAG_BF16) cross_combine_kernel<bf16_t><<<grid, 256, 0, st>>>(a);
    else cross_combine_kernel<f16_t><<<grid, 256, 0, st>>>(a);
    return check_launch("cross_combine");
}

}  // namespace snag
