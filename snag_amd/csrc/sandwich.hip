// The two norms around a block with its gate and its residual in one pass over the rows:
//
//   h = res_scale x + gate * (post_w N(y) + post_b),   z = pre_w N(h) + pre_b,     N = RMS or layer norm
//
// and its backward with every parameter gradient.  Bound by memory: a row of x and y is read and a row of h and z written, once; the
// backward reads x, y, dh, dz and writes dx, dy.  It recomputes h from x and y (the same bytes as a stored h, and exact: a 16-bit h would
// put its rounding into d pre_w), from the four statistics per row the forward saved.  All arithmetic and all sums are fp32, each output is
// rounded once; the variance is taken around the mean (two passes over registers).
//
// TPR threads work on one row (32, 64: lane groups, no LDS; 256, 512: a workgroup) with NU x 4 elements per thread in registers.  In the backward
// a worker walks a run of rows and keeps the parameter gradients of its columns in registers; its run lies inside one gate row or covers
// whole gate rows, the partial sums go to a slab [worker][gradient][dim] and are added up in the workers' order (no atomics).
#include <type_traits>
#include "cross.hip.h"

namespace snag {

struct SandwichArgs {
    const void *x, *y, *post_w, *post_b, *pre_w, *pre_b, *gate;
    int w32, g32;                  // parameters / gate in fp32 (else y's type)
    int64_t row0, rows, rows_per_gate;      // row0: the launch's first row (forward; a launch stays below 2^32 threads)
    int dim, layer;
    float res_scale, eps;
    void *h, *z;
    float* stats;                  // [rows][4]: mean y, 1 / deviation y, mean h, 1 / deviation h (means 0 for RMS)
    // backward
    const void *dh, *dz;           // NULL: zero
    void *dx, *dy, *dgate;
    int dgate_direct;              // every gate row lies inside one worker's run: written by it
    int64_t workers, run, chunks;  // rows per worker; workers per gate row (dgate_direct: 1)
    float* slab;                   // [workers][kGrads][dim]
};
enum { kPostW, kPostB, kPreW, kPreB, kGate, kGrads };

template <class T> struct Four { using vec = __attribute__((ext_vector_type(4))) T; };

// thread t's four elements of step u: neighbours (VEC) or a stride of TPR apart (any dim, any alignment)
template <int TPR, bool VEC> __device__ __forceinline__ int column(int u, int j, int t) { return VEC ? (u * TPR + t) * 4 + j : (u * 4 + j) * TPR + t; }

// a thread's elements of a row as they lie in memory, and as fp32 (0 behind the row's end)
template <class T, int NU> struct Raw { typename Four<T>::vec v[NU]; };
template <class T, int TPR, int NU, bool VEC>
__device__ __forceinline__ Raw<T, NU> raw_row(const T* p, int D, int t) {
    Raw<T, NU> r;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        r.v[u] = typename Four<T>::vec{};
        if constexpr (VEC) {
            const int c = column<TPR, VEC>(u, 0, t);
            if (c < D) r.v[u] = *(const typename Four<T>::vec*)(p + c);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = column<TPR, VEC>(u, j, t);
                if (c < D) r.v[u][j] = p[c];
            }
        }
    }
    return r;
}
template <class T, int NU>
__device__ __forceinline__ void widen(float (&r)[NU][4], const Raw<T, NU>& v) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) r[u][j] = (float)v.v[u][j];
}
template <class T, int TPR, int NU, bool VEC>
__device__ __forceinline__ void load_row(float (&r)[NU][4], const T* p, int D, int t) { widen<T, NU>(r, raw_row<T, TPR, NU, VEC>(p, D, t)); }
template <class T, int TPR, int NU, bool VEC>
__device__ __forceinline__ void store_row(T* p, const float (&r)[NU][4], int D, int t) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        if constexpr (VEC) {
            const int c = column<TPR, VEC>(u, 0, t);
            typename Four<T>::vec v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (T)r[u][j];
            if (c < D) *(typename Four<T>::vec*)(p + c) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = column<TPR, VEC>(u, j, t);
                if (c < D) p[c] = (T)r[u][j];
            }
        }
    }
}
// a parameter row (fp32 or T), `none` where there is none
template <class T, int TPR, int NU, bool VEC>
__device__ __forceinline__ void load_param(float (&r)[NU][4], const void* p, int is32, int64_t row, float none, int D, int t) {
    if (p == nullptr) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) r[u][j] = none;
    } else if (is32) {
        load_row<float, TPR, NU, VEC>(r, (const float*)p + row * D, D, t);
    } else {
        load_row<T, TPR, NU, VEC>(r, (const T*)p + row * D, D, t);
    }
}

// sums over the TPR threads of a row; every thread gets them
constexpr int kMaxWaves = 8;
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float (*red)[kMaxWaves][2], int& turn) {
    if constexpr (TPR == 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = sum16(s[i]), s[i] += __shfl_xor(s[i], 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = sum64(s[i]);
        if constexpr (TPR > 64) {
            // two sets of slots in turn: one barrier per sum
            float (*slot)[2] = red[turn];
            turn ^= 1;
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) slot[wave][i] = s[i];
            }
            // LDS alone has to be visible: global loads may stay in flight across the barrier
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s[i] = slot[0][i];
#pragma unroll
                for (int w = 1; w < TPR / 64; ++w) s[i] += slot[w][i];
            }
        }
    }
}

template <int TPR, int NU, bool VEC>
__device__ __forceinline__ void row_stats(const float (&v)[NU][4], int D, int layer, float eps, int t, float (*red)[kMaxWaves][2], int& turn, float& mean, float& rstd) {
    mean = 0.f;
    if (layer) {
        float s[1] = {0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0] += v[u][j];
        row_sums<TPR, 1>(s, red, turn);
        mean = s[0] / (float)D;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float e = column<TPR, VEC>(u, j, t) < D ? v[u][j] - mean : 0.f;
            s[0] = fmaf(e, e, s[0]);
        }
    row_sums<TPR, 1>(s, red, turn);
    rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
}

// One row a worker: the launch is wide enough to hide its reads (16384 rows of 4096 in bf16 around an fp32 stream: 147 us, 5.5 TB/s).
template <class TX, class TY, int TPR, int NU, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void sandwich_fwd_kernel(SandwichArgs a) {
    __shared__ float red[2][kMaxWaves][2];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const int64_t row = a.row0 + (TPR >= 256 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR);
    if (TPR < 256 && row >= a.rows) return;       // otherwise one row per workgroup
    const int D = a.dim;
    float y[NU][4], x[NU][4], p[NU][4], b[NU][4], g[NU][4];
    load_row<TY, TPR, NU, VEC>(y, (const TY*)a.y + row * D, D, t);
    load_row<TX, TPR, NU, VEC>(x, (const TX*)a.x + row * D, D, t);
    load_param<TY, TPR, NU, VEC>(p, a.post_w, a.w32, 0, 1.f, D, t);
    load_param<TY, TPR, NU, VEC>(b, a.post_b, a.w32, 0, 0.f, D, t);
    load_param<TY, TPR, NU, VEC>(g, a.gate, a.g32, row / a.rows_per_gate, 1.f, D, t);
    float my, ry, mh, rh;
    row_stats<TPR, NU, VEC>(y, D, a.layer, a.eps, t, red, turn, my, ry);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float post = fmaf((y[u][j] - my) * ry, p[u][j], b[u][j]);
            x[u][j] = column<TPR, VEC>(u, j, t) < D ? fmaf(g[u][j], post, a.res_scale * x[u][j]) : 0.f;
        }
    store_row<TX, TPR, NU, VEC>((TX*)a.h + row * D, x, D, t);
    load_param<TY, TPR, NU, VEC>(p, a.pre_w, a.w32, 0, 1.f, D, t);
    load_param<TY, TPR, NU, VEC>(b, a.pre_b, a.w32, 0, 0.f, D, t);
    row_stats<TPR, NU, VEC>(x, D, a.layer, a.eps, t, red, turn, mh, rh);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = fmaf((x[u][j] - mh) * rh, p[u][j], b[u][j]);
    store_row<TY, TPR, NU, VEC>((TY*)a.z + row * D, x, D, t);
    if (t == 0 && a.stats != nullptr) *(f32x4*)(a.stats + row * 4) = f32x4{my, ry, mh, rh};
}

// With up to eight elements a thread the weights and (while it lasts) the gate stay in registers and the next row is in flight while the present
// one is worked on (rows of 4096 in bf16 around an fp32 stream: 340 -> 264 us, 4.6 TB/s); with 16 there is no room for either.
template <class TX, class TY, int TPR, int NU, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void sandwich_bwd_kernel(SandwichArgs a) {
    constexpr bool KEEP = NU <= 2;
    __shared__ float red[2][kMaxWaves][2];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const int64_t worker = TPR >= 256 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (TPR < 256 && worker >= a.workers) return;
    const int D = a.dim;
    // rows of this worker: run `worker % chunks` of gate row `worker / chunks`, or `run` rows anywhere (whole gate rows)
    int64_t r0, r1;
    if (a.dgate_direct) {
        r0 = worker * a.run;
        r1 = min(a.rows, r0 + a.run);
    } else {
        const int64_t group = worker / a.chunks;
        r0 = group * a.rows_per_gate + worker % a.chunks * a.run;
        r1 = min((group + 1) * a.rows_per_gate, r0 + a.run);
    }
    float sum[kGrads][NU][4], pw[NU][4], pb[NU][4], qw[NU][4], g[NU][4];
#pragma unroll
    for (int k = 0; k < kGrads; ++k)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[k][u][j] = 0.f;
    const float inv_d = 1.0f / (float)D;
    Raw<TY, NU> ny, ne;
    Raw<TX, NU> nx, nd;
    f32x4 nst{};
    auto fetch = [&](int64_t row) {
        ny = raw_row<TY, TPR, NU, VEC>((const TY*)a.y + row * D, D, t);
        nx = raw_row<TX, TPR, NU, VEC>((const TX*)a.x + row * D, D, t);
        nd = a.dh != nullptr ? raw_row<TX, TPR, NU, VEC>((const TX*)a.dh + row * D, D, t) : Raw<TX, NU>{};
        ne = a.dz != nullptr ? raw_row<TY, TPR, NU, VEC>((const TY*)a.dz + row * D, D, t) : Raw<TY, NU>{};
        nst = *(const f32x4*)(a.stats + row * 4);
    };
    auto weights = [&]() {
        load_param<TY, TPR, NU, VEC>(pw, a.post_w, a.w32, 0, 1.f, D, t);
        load_param<TY, TPR, NU, VEC>(pb, a.post_b, a.w32, 0, 0.f, D, t);
        load_param<TY, TPR, NU, VEC>(qw, a.pre_w, a.w32, 0, 1.f, D, t);
    };
    if (KEEP && r0 < r1) fetch(r0), weights();
    int64_t grow = r0 < r1 ? r0 / a.rows_per_gate : 0, gate_end = (grow + 1) * a.rows_per_gate;
    bool fresh = true;                                     // the gate row has not been read yet
    for (int64_t row = r0; row < r1; ++row) {
        if (!KEEP) fetch(row), weights();
        if (!KEEP || fresh) load_param<TY, TPR, NU, VEC>(g, a.gate, a.g32, grow, 1.f, D, t), fresh = false;
        float y[NU][4], x[NU][4], d[NU][4], e[NU][4], b[NU][4];
        widen<TY, NU>(y, ny);
        widen<TX, NU>(x, nx);
        widen<TX, NU>(d, nd);
        widen<TY, NU>(e, ne);
        const float my = nst[0], ry = nst[1], mh = nst[2], rh = nst[3];
        if (KEEP && row + 1 < r1) fetch(row + 1);
        // y <- N(y), x <- N(h), b <- post
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[u][j] = (y[u][j] - my) * ry;
                b[u][j] = fmaf(y[u][j], pw[u][j], pb[u][j]);
                x[u][j] = (fmaf(g[u][j], b[u][j], a.res_scale * x[u][j]) - mh) * rh;
            }
        if (a.dz != nullptr) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sum[kPreW][u][j] = fmaf(e[u][j], x[u][j], sum[kPreW][u][j]);
                    sum[kPreB][u][j] += e[u][j];
                    e[u][j] *= qw[u][j];                      // 0 behind the row's end, as dz is
                    s[0] = fmaf(e[u][j], x[u][j], s[0]);
                    s[1] += e[u][j];
                }
            row_sums<TPR, 2>(s, red, turn);
            const float m1 = s[0] * inv_d, m2 = a.layer ? s[1] * inv_d : 0.f;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[u][j] = fmaf(rh, e[u][j] - fmaf(x[u][j], m1, m2), d[u][j]);
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = column<TPR, VEC>(u, j, t) < D;
                x[u][j] = a.res_scale * d[u][j];
                b[u][j] = in ? d[u][j] * b[u][j] : 0.f;       // d gate
                const float dp = in ? d[u][j] * g[u][j] : 0.f;
                sum[kPostW][u][j] = fmaf(dp, y[u][j], sum[kPostW][u][j]);
                sum[kPostB][u][j] += dp;
                sum[kGate][u][j] += b[u][j];
                e[u][j] = dp * pw[u][j];
                s[0] = fmaf(e[u][j], y[u][j], s[0]);
                s[1] += e[u][j];
            }
        store_row<TX, TPR, NU, VEC>((TX*)a.dx + row * D, x, D, t);
        row_sums<TPR, 2>(s, red, turn);
        const float m1 = s[0] * inv_d, m2 = a.layer ? s[1] * inv_d : 0.f;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) e[u][j] = ry * (e[u][j] - fmaf(y[u][j], m1, m2));
        store_row<TY, TPR, NU, VEC>((TY*)a.dy + row * D, e, D, t);
        if (row + 1 == gate_end) {
            if (a.dgate_direct && a.dgate != nullptr) {
                if (a.g32) store_row<float, TPR, NU, VEC>((float*)a.dgate + grow * D, sum[kGate], D, t);
                else store_row<TY, TPR, NU, VEC>((TY*)a.dgate + grow * D, sum[kGate], D, t);
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[kGate][u][j] = 0.f;
            }
            ++grow;
            gate_end += a.rows_per_gate;
            fresh = true;
        }
    }
    float* out = a.slab + worker * kGrads * D;
#pragma unroll
    for (int k = 0; k < kGrads; ++k)
        if (k != kGate || !a.dgate_direct) store_row<float, TPR, NU, VEC>(out + k * D, sum[k], D, t);
}

// sum of v, as a tree
__device__ __forceinline__ float tree16(float (&v)[16]) {
#pragma unroll
    for (int n = 8; n > 0; n >>= 1)
#pragma unroll
        for (int u = 0; u < n; ++u) v[u] += v[u + n];
    return v[0];
}
// Column sums of the slab: y = gradient (0..3: all workers; from 4 on: gate row y - 4, its own workers), 64 columns x 16 runs of workers a workgroup.
// A run of 256 partials one after another costs 2^-24 sqrt(128) of the sum: 16 chains a run, joined by trees (45000 rows of 128: 3.3e-7 -> 1.3e-7; the same time).
struct SandwichSums {
    const float* slab;
    int64_t workers, chunks;
    int dim;
    void* out[4];
    int w32;
    void* dgate;
    int g32;
};
template <class TY>
__global__ __launch_bounds__(1024) void sandwich_sums_kernel(SandwichSums a) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, c = blockIdx.x * 64 + lane, k = min((int)blockIdx.y, (int)kGate);
    const int64_t group = (int64_t)blockIdx.y - kGate;
    void* out = k < kGate ? a.out[k] : a.dgate;
    if (out == nullptr) return;                   // the whole workgroup
    const int64_t w0 = k < kGate ? 0 : group * a.chunks, n = k < kGate ? a.workers : a.chunks, per = (n + 15) / 16;
    const int64_t b0 = w0 + run * per, b1 = min(w0 + n, b0 + per);
    float v[16] = {};
    if (c < a.dim) {
        const float* p = a.slab + (b0 * kGrads + k) * a.dim + c;
        const int64_t step = (int64_t)kGrads * a.dim;
        int64_t i = b0;
        auto add = [&](int at) {
            float w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = p[u * step];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[at + u] += w[u];
            i += 8, p += 8 * step;
        };
        while (i + 16 <= b1) add(0), add(8);
        if (i + 8 <= b1) add(0);
        for (; i < b1; ++i, p += step) v[0] += *p;
    }
    part[run][lane] = tree16(v);
    __syncthreads();
    if (run != 0 || c >= a.dim) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] = part[r][lane];
    const float s = tree16(v);
    if (k < kGate ? a.w32 : a.g32) ((float*)out)[(k < kGate ? 0 : group * a.dim) + c] = s;
    else ((TY*)out)[(k < kGate ? 0 : group * a.dim) + c] = (TY)s;
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// the backward holds eight rows' worth of registers per thread (gradients, weights, the next row): wide rows take 512 threads
static int threads_per_row(int dim) { return dim <= 128 ? 32 : dim <= 512 ? 64 : dim <= 2048 ? 256 : 512; }

struct SandwichPlan { int direct; int64_t workers, run, chunks; };
// Workers: enough to fill the chip (lane groups: 4096; workgroups of 256: 1024, of 512: 512), no more than rows.
static SandwichPlan sandwich_plan(int64_t rows, int64_t rows_per_gate, int dim) {
    const int tpr = threads_per_row(dim);
    const int64_t want = tpr == 512 ? 512 : tpr == 256 ? 1024 : 4096;
    SandwichPlan p{};
    const int64_t share = (rows + want - 1) / want;
    if (rows_per_gate <= share) {
        p.direct = 1, p.chunks = 1;
        p.run = (share + rows_per_gate - 1) / rows_per_gate * rows_per_gate;
        p.workers = (rows + p.run - 1) / p.run;
    } else {
        const int64_t gates = rows / rows_per_gate;
        p.chunks = (rows_per_gate + share - 1) / share;
        p.run = (rows_per_gate + p.chunks - 1) / p.chunks;
        p.chunks = (rows_per_gate + p.run - 1) / p.run;
        p.workers = gates * p.chunks;
    }
    return p;
}

template <class TX, class TY>
static void sandwich_launch(const SandwichArgs& a, int64_t items, bool vec, bool bwd, hipStream_t st) {
    const int tpr = threads_per_row(a.dim);
    const int threads = tpr > 256 ? tpr : 256, per = threads / tpr;
    const dim3 grid((unsigned)((items + per - 1) / per));
#define GO(TPR, NU)                                                                       \
    do {                                                                                  \
        if (bwd) {                                                                        \
            if (vec) sandwich_bwd_kernel<TX, TY, TPR, NU, true><<<grid, threads, 0, st>>>(a); \
            else sandwich_bwd_kernel<TX, TY, TPR, NU, false><<<grid, threads, 0, st>>>(a);    \
        } else {                                                                          \
            if (vec) sandwich_fwd_kernel<TX, TY, TPR, NU, true><<<grid, threads, 0, st>>>(a); \
            else sandwich_fwd_kernel<TX, TY, TPR, NU, false><<<grid, threads, 0, st>>>(a);    \
        }                                                                                 \
    } while (0)
    const int D = a.dim;
    if (D <= 128) GO(32, 1);
    else if (D <= 256) GO(64, 1);
    else if (D <= 512) GO(64, 2);
    else if (D <= 1024) GO(256, 1);
    else if (D <= 2048) GO(256, 2);
    else if (D <= 4096) GO(512, 2);
    else GO(512, 4);
#undef GO
}

static int sandwich_check(const void* x, int x_dtype, const void* y, int y_dtype, int64_t rows, int dim, int w_dtype, const void* gate, int gate_dtype, int64_t rows_per_gate, int kind) {
    SNAG_REQUIRE(y_dtype == SNAG_F32 || y_dtype == SNAG_BF16 || y_dtype == SNAG_F16, SNAG_ERR_ARG, "sandwich norm: dtype %d", y_dtype);
    SNAG_REQUIRE(x_dtype == y_dtype || x_dtype == SNAG_F32, SNAG_ERR_UNSUPPORTED, "sandwich norm: the residual stream is fp32 or of the block output's type");
    SNAG_REQUIRE(w_dtype == y_dtype || w_dtype == SNAG_F32, SNAG_ERR_UNSUPPORTED, "sandwich norm: weights and biases are fp32 or of the block output's type");
    SNAG_REQUIRE(gate == nullptr || gate_dtype == y_dtype || gate_dtype == SNAG_F32, SNAG_ERR_UNSUPPORTED, "sandwich norm: the gate is fp32 or of the block output's type");
    SNAG_REQUIRE(rows >= 0 && dim >= 1, SNAG_ERR_ARG, "sandwich norm: %lld rows of %d", (long long)rows, dim);
    SNAG_REQUIRE(dim <= SNAG_SANDWICH_MAX_DIM, SNAG_ERR_UNSUPPORTED, "sandwich norm: row width %d > %d", dim, SNAG_SANDWICH_MAX_DIM);
    SNAG_REQUIRE(rows < (int64_t)1 << 31, SNAG_ERR_UNSUPPORTED, "sandwich norm: %lld rows", (long long)rows);
    SNAG_REQUIRE(kind == SNAG_NORM_RMS || kind == SNAG_NORM_LAYER, SNAG_ERR_ARG, "sandwich norm: kind %d", kind);
    SNAG_REQUIRE(gate == nullptr || (rows_per_gate >= 1 && rows % rows_per_gate == 0), SNAG_ERR_ARG, "sandwich norm: %lld rows are not a multiple of %lld rows per gate", (long long)rows,
                 (long long)rows_per_gate);
    SNAG_REQUIRE(rows == 0 || (x != nullptr && y != nullptr), SNAG_ERR_ARG, "sandwich norm: null x / y");
    return SNAG_OK;
}
static size_t bytes_of(int dtype) { return dtype == SNAG_F32 ? 4 : 2; }
static bool aligned4(const void* p, int dtype) { return ((uintptr_t)p & (4 * bytes_of(dtype) - 1)) == 0; }

// items: rows of this launch (forward) or workers
static void sandwich_go(const SandwichArgs& a, int64_t items, int x_dtype, int y_dtype, bool vec, bool bwd, hipStream_t st) {
    if (y_dtype == SNAG_F32) sandwich_launch<float, float>(a, items, vec, bwd, st);
    else if (y_dtype == SNAG_BF16) x_dtype == SNAG_F32 ? sandwich_launch<float, bf16_t>(a, items, vec, bwd, st) : sandwich_launch<bf16_t, bf16_t>(a, items, vec, bwd, st);
    else x_dtype == SNAG_F32 ? sandwich_launch<float, f16_t>(a, items, vec, bwd, st) : sandwich_launch<f16_t, f16_t>(a, items, vec, bwd, st);
}

}  // namespace snag

using namespace snag;

extern "C" SNAG_API int snag_sandwich_fwd(const void* x, int x_dtype, const void* y, int y_dtype, int64_t rows, int dim, const void* post_w, const void* post_b,
                                          const void* pre_w, const void* pre_b, int w_dtype, const void* gate, int gate_dtype, int64_t rows_per_gate,
                                          float res_scale, int kind, float eps, void* h, void* z, float* stats, void* stream) {
    if (int rc = sandwich_check(x, x_dtype, y, y_dtype, rows, dim, w_dtype, gate, gate_dtype, rows_per_gate, kind)) return rc;
    if (rows == 0) return SNAG_OK;
    SNAG_REQUIRE(h != nullptr && z != nullptr, SNAG_ERR_ARG, "sandwich norm: null h / z");
    SNAG_REQUIRE(stats == nullptr || ((uintptr_t)stats & 15) == 0, SNAG_ERR_ARG, "sandwich norm: stats are not 16-byte aligned");
    SandwichArgs a{};
    a.x = x, a.y = y, a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w, a.pre_b = pre_b, a.gate = gate;
    a.w32 = w_dtype == SNAG_F32, a.g32 = gate_dtype == SNAG_F32;
    a.rows = rows, a.rows_per_gate = gate != nullptr ? rows_per_gate : rows, a.dim = dim, a.layer = kind == SNAG_NORM_LAYER, a.res_scale = res_scale, a.eps = eps;
    a.h = h, a.z = z, a.stats = stats;
    const bool vec = dim % 4 == 0 && aligned4(x, x_dtype) && aligned4(y, y_dtype) && aligned4(h, x_dtype) && aligned4(z, y_dtype) && aligned4(post_w, w_dtype) &&
                     aligned4(post_b, w_dtype) && aligned4(pre_w, w_dtype) && aligned4(pre_b, w_dtype) && aligned4(gate, gate_dtype);
    constexpr int64_t kRows = (int64_t)1 << 22;                // of up to 512 threads
    for (; a.row0 < rows; a.row0 += kRows) {
        sandwich_go(a, rows - a.row0 < kRows ? rows - a.row0 : kRows, x_dtype, y_dtype, vec, false, (hipStream_t)stream);
        if (int rc = check_launch("sandwich_fwd")) return rc;
    }
    return SNAG_OK;
}

extern "C" SNAG_API int64_t snag_sandwich_work_floats(int64_t rows, int64_t rows_per_gate, int dim) {
    if (rows <= 0 || rows_per_gate < 1 || dim < 1) return 0;
    return sandwich_plan(rows, rows_per_gate, dim).workers * kGrads * dim;
}

extern "C" SNAG_API int snag_sandwich_bwd(const void* x, int x_dtype, const void* y, int y_dtype, int64_t rows, int dim, const void* post_w, const void* post_b,
                                          const void* pre_w, int w_dtype, const void* gate, int gate_dtype, int64_t rows_per_gate, float res_scale, int kind,
                                          const float* stats, const void* d_h, const void* d_z, void* d_x, void* d_y, void* d_post_w, void* d_post_b,
                                          void* d_pre_w, void* d_pre_b, void* d_gate, float* work, int64_t work_floats, void* stream) {
    if (int rc = sandwich_check(x, x_dtype, y, y_dtype, rows, dim, w_dtype, gate, gate_dtype, rows_per_gate, kind)) return rc;
    SNAG_REQUIRE(gate != nullptr || d_gate == nullptr, SNAG_ERR_ARG, "sandwich norm backward: d_gate without a gate");
    SandwichArgs a{};
    const int64_t rpg = gate != nullptr ? rows_per_gate : (rows > 0 ? rows : 1);
    SNAG_REQUIRE(rows == 0 || (stats != nullptr && d_x != nullptr && d_y != nullptr), SNAG_ERR_ARG, "sandwich norm backward: null stats / d_x / d_y");
    SNAG_REQUIRE(((uintptr_t)stats & 15) == 0, SNAG_ERR_ARG, "sandwich norm backward: stats are not 16-byte aligned");
    SandwichPlan p{};
    if (rows > 0) p = sandwich_plan(rows, rpg, dim);
    SNAG_REQUIRE(rows == 0 || (work != nullptr && work_floats >= p.workers * kGrads * dim), SNAG_ERR_ARG, "sandwich norm backward: workspace of %lld floats, %lld needed",
                 (long long)work_floats, (long long)(p.workers * kGrads * dim));
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        a.x = x, a.y = y, a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w, a.gate = gate;
        a.w32 = w_dtype == SNAG_F32, a.g32 = gate_dtype == SNAG_F32;
        a.rows = rows, a.rows_per_gate = rpg, a.dim = dim, a.layer = kind == SNAG_NORM_LAYER, a.res_scale = res_scale;
        a.stats = (float*)stats, a.dh = d_h, a.dz = d_z, a.dx = d_x, a.dy = d_y, a.dgate = d_gate;
        a.dgate_direct = p.direct, a.workers = p.workers, a.run = p.run, a.chunks = p.chunks, a.slab = work;
        const bool vec = dim % 4 == 0 && aligned4(x, x_dtype) && aligned4(y, y_dtype) && aligned4(post_w, w_dtype) && aligned4(post_b, w_dtype) &&
                         aligned4(pre_w, w_dtype) && aligned4(gate, gate_dtype) && aligned4(d_h, x_dtype) && aligned4(d_z, y_dtype) && aligned4(d_x, x_dtype) &&
                         aligned4(d_y, y_dtype) && aligned4(d_gate, gate_dtype) && aligned16(work);
        sandwich_go(a, a.workers, x_dtype, y_dtype, vec, true, st);
        if (int rc = check_launch("sandwich_bwd")) return rc;
    }
    if (d_post_w == nullptr && d_post_b == nullptr && d_pre_w == nullptr && d_pre_b == nullptr && d_gate == nullptr) return SNAG_OK;
    SandwichSums s{};
    s.slab = work, s.workers = p.workers, s.chunks = p.chunks, s.dim = dim;
    s.out[kPostW] = d_post_w, s.out[kPostB] = d_post_b, s.out[kPreW] = d_pre_w, s.out[kPreB] = d_pre_b;
    s.w32 = w_dtype == SNAG_F32, s.g32 = gate_dtype == SNAG_F32;
    const int64_t gates = d_gate != nullptr && rows > 0 && !p.direct ? rows / rpg : 0;
    s.dgate = gates > 0 ? d_gate : nullptr;
    SNAG_REQUIRE(gates + kGate <= 65535, SNAG_ERR_UNSUPPORTED, "sandwich norm backward: %lld gate rows", (long long)gates);
    const dim3 grid((unsigned)((dim + 63) / 64), (unsigned)(kGate + gates));
    if (y_dtype == SNAG_F32) sandwich_sums_kernel<float><<<grid, 1024, 0, st>>>(s);
    else if (y_dtype == SNAG_BF16) sandwich_sums_kernel<bf16_t><<<grid, 1024, 0, st>>>(s);
    else sandwich_sums_kernel<f16_t><<<grid, 1024, 0, st>>>(s);
    return check_launch("sandwich_sums");
}
