// Cross attention: the choice of a path, the checks of arguments and the C entries.
#include "cross.hip.h"

namespace snag {

static int elem_size(int dtype) { return dtype == SNAG_F32 ? 4 : 2; }

// Workgroups that run at a time: two of four waves on a CU, or four waves on their own, one per SIMD -- two per SIMD where their registers allow
// (the kernels' launch bounds): 16-bit forward, and backward up to 64 elements a head.  64 sequences x 8 heads of 64 in bf16 with 8 rows over
// 4096 keys, ranges for 512 / 1024 / 2048 workgroups: 250 / 162 / 128 us; with 16 rows in fp32 512 / 271 / 275.
static int slots(int waves, int dtype, int dp, bool backward) {
    if (waves > 1) return 2 * 256;
    return dtype != SNAG_F32 && (!backward || dp <= 64) ? 8 * 256 : 4 * 256;
}
// How many ranges a loop over `n` keys or rows is cut into when `groups` workgroups exist without cutting.  In units of 64 keys' or rows' time (1 - 3
// us): a round of workgroups takes 5 to start and end besides its loop, joining ranges 4 and 0.5 for each (a launch, the partial results).  Both
// sides: 192 groups over 4096 rows of 128: 2 ranges 154 us, 3 181; 92 groups over 316 keys: 1 range 17, 2 24; 72 groups over 777 keys: 1 range
// 46, 5 32, 12 40.  At least 128 keys or rows a range.
static int ranges_for(int64_t groups, int64_t n, int64_t slots) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; groups > 0 && groups < slots && s <= 64 && (s == 1 || s <= n / 128); ++s) {
        const double cost = (double)((groups * s + slots - 1) / slots) * (5 + (double)n / 64 / s) + (s > 1 ? 4 + 0.5 * s : 0);
        if (cost < least) least = cost, best = s;
    }
    return best;
}

// rows_path: a few rows per key/value head (csrc/cross_rows.hip) -- a 32-row product would multiply mostly padding.  Up to 4 rows; up to 8 in fp32,
// whose matrix instructions are 16 times slower (heads of 128, 512 problems over 4096 keys, here / in tiles: 5 rows 438 / 590 us, 8 rows 632 / 580;
// 64 problems backward: 5 rows 125 / 470, 8 rows 138 / 470).  16 bit, 8 rows in tiles: 234 us, 4.6 TB/s of keys.
// One wave a workgroup where 32 rows (keys) are all there is; four otherwise, and for the backward of fp32 rows over 64, whose tiles do not fit
// one wave's registers.
static CrossPlan cross_plan(int dtype, int B, int Lq, int Lk, int H, int Hkv, int d) {
    CrossPlan p{};
    const int64_t rows = (int64_t)Lq * (H / Hkv), bh = (int64_t)B * Hkv;
    p.dp = d <= 32 ? 32 : d <= 64 ? 64 : 128;
    const bool wide = dtype == SNAG_F32 && p.dp == 128;
    p.nw_fwd = rows > 32 ? 4 : 1;
    p.nw_dq = rows > 32 || wide ? 4 : 1;
    p.nw_k = Lk > 32 || wide ? 4 : 1;
    p.rows_path = rows <= (dtype == SNAG_F32 ? 8 : 4);
    if (p.rows_path) {
        p.s_fwd = p.s_dq = cross_rows_splits(B, Hkv, Lk, d, dtype);
        p.s_dkv = 1;
        return p;
    }
    p.s_fwd = ranges_for(bh * ((rows + p.nw_fwd * 32 - 1) / (p.nw_fwd * 32)), Lk, slots(p.nw_fwd, dtype, p.dp, false));
    p.s_dq = ranges_for(bh * ((rows + p.nw_dq * 32 - 1) / (p.nw_dq * 32)), Lk, slots(p.nw_dq, dtype, p.dp, true));
    p.s_dkv = ranges_for(bh * ((Lk + p.nw_k * 32 - 1) / (p.nw_k * 32)), rows, slots(p.nw_k, dtype, p.dp, true));
    return p;
}

static int64_t stat_floats(const CrossPlan& p, int B, int Lq, int H, int Hkv) { return p.rows_path ? 0 : 2 * (int64_t)B * Hkv * padded_rows(Lq * (H / Hkv)); }
static int64_t fwd_part_floats(const CrossPlan& p, int64_t n, int d) { return p.s_fwd > 1 ? p.s_fwd * n * (d + 2) : 0; }
static int64_t bwd_part_floats(const CrossPlan& p, int64_t nq, int64_t nk, int d) {
    const int64_t dq = p.s_dq > 1 ? p.s_dq * nq * d : 0, dkv = p.s_dkv > 1 ? 2 * p.s_dkv * nk * d : 0;
    return dq > dkv ? dq : dkv;
}

static int cross_shapes(int dtype, int B, int Lq, int Lk, int H, int Hkv, int d) {
    SNAG_REQUIRE(dtype == SNAG_F32 || dtype == SNAG_BF16 || dtype == SNAG_F16, SNAG_ERR_ARG, "cross attention: dtype %d", dtype);
    SNAG_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && H >= 1 && Hkv >= 1, SNAG_ERR_ARG, "cross attention: negative or empty size (B %d, Lq %d, Lk %d, H %d, Hkv %d)", B, Lq, Lk, H, Hkv);
    SNAG_REQUIRE(H % Hkv == 0, SNAG_ERR_ARG, "cross attention: %d heads are not a multiple of %d key/value heads", H, Hkv);
    SNAG_REQUIRE(d >= 1 && d <= SNAG_CROSS_MAX_HEAD_DIM, SNAG_ERR_UNSUPPORTED, "cross attention: head dimension %d is not in 1..%d", d, SNAG_CROSS_MAX_HEAD_DIM);
    const int64_t G = H / Hkv;
    SNAG_REQUIRE(G <= 65535 && (int64_t)Lq * G <= (1 << 30) && Lk <= (1 << 30), SNAG_ERR_UNSUPPORTED, "cross attention: more than 2^30 rows or keys in one problem");
    SNAG_REQUIRE((int64_t)Lq * G * G < (int64_t)1 << 32, SNAG_ERR_UNSUPPORTED, "cross attention: Lq (H / Hkv)^2 = %lld is not below 2^32", (long long)((int64_t)Lq * G * G));
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
    // ceil(2^32 / G) as a multiplier is exact for rows below 2^32 / (its excess over 2^32 / G, times G), and that is below G
    a.g_magic = a.G > 1 ? (uint32_t)((((uint64_t)1 << 32) + a.G - 1) / a.G) : 0;
    a.g_one = a.G > 1 ? 0 : ~0u;
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
    return backward ? stat_floats(p, B, Lq, H, Hkv) + bwd_part_floats(p, nq, nk, d) : fwd_part_floats(p, nq, d);
}

extern "C" SNAG_API int snag_cross_fwd(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int d,
                                       const int64_t* strides_host, const void* kv_lens, int lens_bytes, const uint8_t* key_mask, int64_t mask_ld, float scale,
                                       void* out, void* out_lo, float* lse, float* work, int64_t work_floats, void* stream) {
    CrossArgs a{};
    if (int rc = cross_args(a, q, k, v, dtype, B, Lq, Lk, H, Hkv, d, strides_host, kv_lens, lens_bytes, key_mask, mask_ld, scale)) return rc;
    if (B == 0 || Lq == 0) return SNAG_OK;
    SNAG_REQUIRE(out != nullptr && lse != nullptr, SNAG_ERR_ARG, "cross attention: null out / lse");
    const CrossPlan p = cross_plan(dtype, B, Lq, Lk, H, Hkv, d);
    const int64_t need = snag_cross_work_floats(dtype, B, Lq, Lk, H, Hkv, d, 0);
    SNAG_REQUIRE(need == 0 || (work != nullptr && work_floats >= need), SNAG_ERR_ARG, "cross attention: workspace of %lld floats, %lld needed", (long long)work_floats, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    a.out = out, a.out_lo = out_lo, a.lse = lse, a.part = work, a.splits = p.s_fwd;
    a.vec_o = d % (16 / elem_size(dtype)) == 0 && aligned16(out) && aligned16(out_lo);
    a.per_split = range_of(Lk, a.splits);
    const int rc = p.rows_path ? cross_rows_fwd(a, dtype, st) : cross_tiles_fwd(a, p, dtype, st);
    return rc != SNAG_OK || a.splits == 1 ? rc : cross_combine(a, dtype, st);
}

extern "C" SNAG_API int snag_cross_bwd(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int d,
                                       const int64_t* strides_host, const void* kv_lens, int lens_bytes, const uint8_t* key_mask, int64_t mask_ld, float scale,
                                       const void* out, const void* out_lo, const float* lse, const void* d_out, void* d_q, void* d_k, void* d_v,
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
    a.o = out, a.o_lo = out_lo, a.lse = (float*)lse, a.dout = d_out, a.dq = d_q, a.dk = d_k, a.dv = d_v;
    a.vec_o = d % (16 / elem_size(dtype)) == 0 && aligned16(out) && aligned16(out_lo) && aligned16(d_out) && aligned16(d_q) && aligned16(d_k) && aligned16(d_v);
    a.part = work + stat_floats(p, B, Lq, H, Hkv);
    if (p.rows_path && Lq > 0) {
        a.splits = p.s_dq;
        if (int rc = cross_rows_bwd(a, dtype, st)) return rc;
        return a.splits == 1 ? SNAG_OK : cross_sum(a.part, (int64_t)B * Lq * H * d, a.splits, d_q, dtype, st);
    }
    CrossPlan pb = p;
    if (p.rows_path) pb.s_dq = pb.s_dkv = 1;               // no rows: d k = d v = 0
    return cross_tiles_bwd(a, pb, work, dtype, st);
}
