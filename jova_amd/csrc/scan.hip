// Selective state space scan over time-major sequences.  Per batch element b, channel d and state n:
//   e[t] = dt[t] + bias, or its softplus          h[t] = exp(e[t] A) h[t-1] + e[t] x[t] B[t]
//   y[t] = (sum_n C[t] h[t] + D x[t]) silu(z[t])  (D and z optional)
// B and C are shared by the channels of a group.  Adjoint, with g[t] = dy[t] silu(z[t]):
//   q[t] = C[t] g[t] + exp(e[t+1] A) q[t+1]       dC[t] = sum_d g h        dB[t] = sum_d q e x      dx = g D + e sum_n q B
//   de   = sum_n q exp(e A) h[t-1] A + x sum_n q B                        dA = sum_t q exp(e A) h[t-1] e
//
// Layout: four neighbouring lanes (a quad) share a channel and hold a quarter of its states each (NS of them, padded with
// states that stay zero), so a wave covers 16 channels.  Time goes in tiles of KT steps; within four steps lane q of a quad
// loads, and later stores, step 4j + q, and the quad passes scalars around with quad_perm, which costs nothing extra.
#include "seq.h"

#include <type_traits>

namespace {

constexpr int WAVES = 4, CH = 16 * WAVES;              // channels of a workgroup
template <int NS> struct Tile { static constexpr int KT = NS <= 4 ? 16 : 8; };      // steps between saved states

struct ScanArgs {
    const void *x, *dt, *B, *C, *z, *dy;
    const float *A, *D, *bias, *state0, *dstate_out;
    void *y, *dx, *ddt, *dz;
    float *state_out, *dstate0;
    float* ckpt;                                       // [tiles][batch][d][4 NS]: the state in front of every tile
    float *part_bc, *part_a, *part_d;                  // partial sums of dB | dC, dA, dD | dbias
    const int* lengths;
    long long x_t, x_b, dt_t, dt_b, z_t, z_b, B_t, B_b, B_g, C_t, C_b, C_g, dy_t, dy_b;
    long long steps;
    int batch, d, groups, n, softplus;
};

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int I> __device__ __forceinline__ float quad_bcast(float v) { return dpp<I * 0x55>(v); }
__device__ __forceinline__ float quad_xor1(float v) { return dpp<0xB1>(v); }
__device__ __forceinline__ float quad_xor2(float v) { return dpp<0x4E>(v); }
__device__ __forceinline__ float quad_sum(float v) {
    v += quad_xor1(v);
    return v + quad_xor2(v);
}
// p[i] of the four lanes of a quad -> lane q gets the sum of p[q]
__device__ __forceinline__ float quad_scatter_sum(const float* p, bool b0, bool b1) {
    const float r0 = (b0 ? p[1] : p[0]) + quad_xor1(b0 ? p[0] : p[1]);
    const float r1 = (b0 ? p[3] : p[2]) + quad_xor1(b0 ? p[2] : p[3]);
    return (b1 ? r1 : r0) + quad_xor2(b1 ? r0 : r1);
}

struct Where {
    int b, g, ch, q, tile;                             // channel (global), lane of the quad, channel tile of the group
    bool live;                                         // the channel exists
    long long len;
};
__device__ __forceinline__ Where where(const ScanArgs& a) {
    Where w;
    const int dg = a.d / a.groups, tiles = (dg + CH - 1) / CH;
    w.g = blockIdx.x / tiles;
    w.tile = blockIdx.x % tiles;
    w.b = blockIdx.y;
    w.q = threadIdx.x & 3;
    const int c = w.tile * CH + (threadIdx.x >> 2);
    w.live = c < dg;
    w.ch = w.g * dg + (w.live ? c : 0);
    long long n = a.lengths ? a.lengths[w.b] : a.steps;
    w.len = n < 0 ? 0 : n > a.steps ? a.steps : n;
    return w;
}

template <typename T> __device__ __forceinline__ float at_step(const void* p, long long s_t, long long s_b, long long t, const Where& w) {
    return (p && w.live && t < w.len) ? to_f(((const T*)p)[t * s_t + w.b * s_b + w.ch]) : 0.f;
}

// rows of B and C of KT steps -> LDS, fp32, zero behind the sequence and in the padded states
template <typename T, int NS>
struct Rows {
    static constexpr int KT = Tile<NS>::KT, NP = 4 * NS, PER = (2 * KT * NP + 255) / 256;
    float v[PER];
    __device__ __forceinline__ void load(const ScanArgs& a, const Where& w, long long t0) {
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int i = threadIdx.x + 256 * r, n = i % NP, t = (i / NP) % KT;
            v[r] = 0.f;
            if (i >= 2 * KT * NP || n >= a.n || t0 + t >= w.len) continue;
            v[r] = i < KT * NP ? to_f(((const T*)a.B)[(t0 + t) * a.B_t + w.b * a.B_b + w.g * a.B_g + n])
                               : to_f(((const T*)a.C)[(t0 + t) * a.C_t + w.b * a.C_b + w.g * a.C_g + n]);
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (threadIdx.x + 256 * r < 2 * KT * NP) lds[threadIdx.x + 256 * r] = v[r];
    }
};

template <int NS> __device__ __forceinline__ void load_state(const float* p, const ScanArgs& a, const Where& w, float* h) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        h[k] = (p && w.live && n < a.n) ? p[((long long)w.b * a.d + w.ch) * a.n + n] : 0.f;
    }
}
template <int NS> __device__ __forceinline__ void store_state(float* p, const ScanArgs& a, const Where& w, const float* h) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        if (p && w.live && n < a.n) p[((long long)w.b * a.d + w.ch) * a.n + n] = h[k];
    }
}
template <int NS> __device__ __forceinline__ long long ckpt_at(const ScanArgs& a, const Where& w, long long tile) {
    return (((tile * a.batch + w.b) * a.d + w.ch) * 4 + w.q) * NS;
}

template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_fwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS;
    __shared__ __align__(16) float rows[2 * KT * NP];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2;
    float A2[NS], h[NS];
    load_state<NS>(a.state0, a, w, h);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        A2[k] = (w.live && n < a.n) ? a.A[(long long)w.ch * a.n + n] * LOG2E_F : 0.f;
    }
    const float Dv = (a.D && w.live) ? a.D[w.ch] : 0.f, bias = (a.bias && w.live) ? a.bias[w.ch] : 0.f;
    Rows<T, NS> next;
    for (long long t0 = 0; t0 < a.steps; t0 += KT) {
        next.load(a, w, t0);
        float x[KT / 4], e[KT / 4], z[KT / 4];
#pragma unroll
        for (int j = 0; j < KT / 4; ++j) {
            const long long t = t0 + 4 * j + w.q;
            x[j] = at_step<T>(a.x, a.x_t, a.x_b, t, w);
            const float raw = at_step<T>(a.dt, a.dt_t, a.dt_b, t, w) + bias;
            e[j] = t < w.len ? (a.softplus ? softplus_f(raw) : raw) : 0.f;
            z[j] = at_step<T>(a.z, a.z_t, a.z_b, t, w);
        }
        __syncthreads();                               // the tile before has read its rows
        next.put(rows);
        __syncthreads();
        if (a.ckpt && w.live)
#pragma unroll
            for (int k = 0; k < NS; ++k) a.ckpt[ckpt_at<NS>(a, w, t0 / KT) + k] = h[k];
#pragma unroll
        for (int j = 0; j < KT / 4; ++j) {
            float p[4];
            const float u = e[j] * x[j];
            auto step = [&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const float ei = quad_bcast<i>(e[j]), ui = quad_bcast<i>(u);
                const float *Bt = rows + (4 * j + i) * NP + w.q * NS, *Ct = Bt + KT * NP;
                p[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    h[k] = fmaf(__builtin_amdgcn_exp2f(ei * A2[k]), h[k], ui * Bt[k]);
                    p[i] = fmaf(Ct[k], h[k], p[i]);
                }
            };
            step(std::integral_constant<int, 0>());
            step(std::integral_constant<int, 1>());
            step(std::integral_constant<int, 2>());
            step(std::integral_constant<int, 3>());
            float y = fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1));
            if (a.z) y *= z[j] * sigmoid_f(z[j]);
            const long long t = t0 + 4 * j + w.q;
            if (w.live && t < a.steps) ((T*)a.y)[(t * a.batch + w.b) * (long long)a.d + w.ch] = from_f<T>(t < w.len ? y : 0.f);
        }
    }
    store_state<NS>(a.state_out, a, w, h);
}

template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_bwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS;
    __shared__ __align__(16) float rows[2 * KT * NP];
    __shared__ float red[WAVES][KT][2][NP];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float A2[NS], q[NS], dA[NS], dD = 0.f, db = 0.f;
    load_state<NS>(a.dstate_out, a, w, q);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        A2[k] = (w.live && n < a.n) ? a.A[(long long)w.ch * a.n + n] * LOG2E_F : 0.f;
        dA[k] = 0.f;
    }
    const float Dv = (a.D && w.live) ? a.D[w.ch] : 0.f, bias = (a.bias && w.live) ? a.bias[w.ch] : 0.f;
    const int dg_tiles = (a.d / a.groups + CH - 1) / CH;
    (void)dg_tiles;
    for (long long tile = (a.steps + KT - 1) / KT - 1; tile >= 0; --tile) {
        const long long t0 = tile * KT;
        Rows<T, NS> next;
        next.load(a, w, t0);
        float x[KT / 4], e[KT / 4], z[KT / 4], raw[KT / 4], dy[KT / 4], g[KT / 4];
        float h0[NS], hs[KT][NS], as[KT][NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) h0[k] = w.live ? a.ckpt[ckpt_at<NS>(a, w, tile) + k] : 0.f;
#pragma unroll
        for (int j = 0; j < KT / 4; ++j) {
            const long long t = t0 + 4 * j + w.q;
            x[j] = at_step<T>(a.x, a.x_t, a.x_b, t, w);
            raw[j] = at_step<T>(a.dt, a.dt_t, a.dt_b, t, w) + bias;
            e[j] = t < w.len ? (a.softplus ? softplus_f(raw[j]) : raw[j]) : 0.f;
            z[j] = at_step<T>(a.z, a.z_t, a.z_b, t, w);
            dy[j] = at_step<T>(a.dy, a.dy_t, a.dy_b, t, w);
        }
        next.put(rows);
        __syncthreads();
        // the tile's states once more, and the output in front of the gate
#pragma unroll
        for (int j = 0; j < KT / 4; ++j) {
            float p[4];
            const float u = e[j] * x[j];
            auto step = [&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = 4 * j + i;
                const float ei = quad_bcast<i>(e[j]), ui = quad_bcast<i>(u);
                const float *Bt = rows + t * NP + w.q * NS, *Ct = Bt + KT * NP;
                p[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    as[t][k] = __builtin_amdgcn_exp2f(ei * A2[k]);
                    hs[t][k] = fmaf(as[t][k], t > 0 ? hs[t > 0 ? t - 1 : 0][k] : h0[k], ui * Bt[k]);
                    p[i] = fmaf(Ct[k], hs[t][k], p[i]);
                }
            };
            step(std::integral_constant<int, 0>());
            step(std::integral_constant<int, 1>());
            step(std::integral_constant<int, 2>());
            step(std::integral_constant<int, 3>());
            const float pre = fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1));
            g[j] = dy[j];
            if (a.z) {
                const float s = sigmoid_f(z[j]);
                g[j] = dy[j] * z[j] * s;
                const long long t = t0 + 4 * j + w.q;
                if (w.live && t < a.steps)
                    ((T*)a.dz)[(t * a.batch + w.b) * (long long)a.d + w.ch] =
                        from_f<T>(t < w.len ? dy[j] * pre * s * (1.f + z[j] * (1.f - s)) : 0.f);
            }
            dD = fmaf(g[j], x[j], dD);
        }
        float dAt[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) dAt[k] = 0.f;
#pragma unroll
        for (int j = KT / 4 - 1; j >= 0; --j) {
            float pb[4], pf[4];
            const float u = e[j] * x[j];
            auto step = [&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = 4 * j + i;
                const float gi = quad_bcast<i>(g[j]), ui = quad_bcast<i>(u), ei = quad_bcast<i>(e[j]);
                const float *Bt = rows + t * NP + w.q * NS, *Ct = Bt + KT * NP;
                pb[i] = pf[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    q[k] = fmaf(Ct[k], gi, q[k]);
                    pb[i] = fmaf(q[k], Bt[k], pb[i]);
                    float vb = q[k] * ui, vc = gi * hs[t][k];
                    const float wq = q[k] * as[t][k], f = wq * (t > 0 ? hs[t > 0 ? t - 1 : 0][k] : h0[k]);
                    dAt[k] = fmaf(f, ei, dAt[k]);
                    pf[i] = fmaf(f, A2[k], pf[i]);
                    q[k] = wq;
#pragma unroll
                    for (int o = 4; o < 64; o <<= 1) {                   // over the wave's 16 channels
                        vb += __shfl_xor(vb, o, 64);
                        vc += __shfl_xor(vc, o, 64);
                    }
                    if (lane < 4) {
                        red[wave][t][0][lane * NS + k] = vb;
                        red[wave][t][1][lane * NS + k] = vc;
                    }
                }
            };
            step(std::integral_constant<int, 3>());
            step(std::integral_constant<int, 2>());
            step(std::integral_constant<int, 1>());
            step(std::integral_constant<int, 0>());
            const float qb = quad_scatter_sum(pb, b0, b1), fa = quad_scatter_sum(pf, b0, b1) * LN2_F;
            const long long t = t0 + 4 * j + w.q;
            float de = fmaf(qb, x[j], fa);
            if (a.softplus) de *= sigmoid_f(raw[j]);
            if (t >= w.len) de = 0.f;
            db += de;
            if (w.live && t < a.steps) {
                const long long at = (t * a.batch + w.b) * (long long)a.d + w.ch;
                ((T*)a.dx)[at] = from_f<T>(t < w.len ? fmaf(g[j], Dv, qb * e[j]) : 0.f);
                ((T*)a.ddt)[at] = from_f<T>(de);
            }
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) dA[k] += dAt[k];
        __syncthreads();
        for (int i = threadIdx.x; i < KT * 2 * NP; i += 256) {
            const int t = i / (2 * NP);
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) s += (&red[v][0][0][0])[i];
            if (t0 + t < a.steps)
                a.part_bc[((((long long)w.tile * a.steps + t0 + t) * a.batch + w.b) * a.groups + w.g) * 2 * NP + i % (2 * NP)] = s;
        }
    }
    store_state<NS>(a.dstate0, a, w, q);
    dD = quad_sum(dD);
    db = quad_sum(db);
    if (w.live) {
        const long long row = (long long)w.b * a.d + w.ch;
#pragma unroll
        for (int k = 0; k < NS; ++k) a.part_a[row * NP + w.q * NS + k] = dA[k];
        if (w.q == 0) {
            a.part_d[row * 2] = dD;
            a.part_d[row * 2 + 1] = db;
        }
    }
}

// dB, dC [t][b][g][n] from the channel tiles' partial sums, in tile order
template <typename T>
__global__ void __launch_bounds__(256)
scan_fold_bc_kernel(const float* __restrict__ part, long long rows, int tiles, int np, int n, T* __restrict__ dB, T* __restrict__ dC) {
    const long long total = rows * 2 * np;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int col = (int)(i % (2 * np)), k = col % np;
        if (k >= n) continue;
        float s = 0.f;
        for (int t = 0; t < tiles; ++t) s += part[t * total + i];
        (col < np ? dB : dC)[(i / (2 * np)) * n + k] = from_f<T>(s);
    }
}
// dA [d][n], dD [d], dbias [d]: sums over the rows (batch elements), in row order, fp64
__global__ void __launch_bounds__(256)
scan_fold_params_kernel(const float* __restrict__ pa, const float* __restrict__ pd, int rows, int d, int np, int n, float* __restrict__ dA,
                        float* __restrict__ dD, float* __restrict__ db) {
    const long long cols = (long long)d * (np + 2);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < cols; i += (long long)gridDim.x * 256) {
        double s = 0.0;
        if (i < (long long)d * np) {
            if (i % np >= n) continue;
            for (int r = 0; r < rows; ++r) s += (double)pa[(long long)r * d * np + i];
            dA[(i / np) * n + i % np] = (float)s;
        } else {
            const long long j = i - (long long)d * np;
            for (int r = 0; r < rows; ++r) s += (double)pd[(long long)r * d * 2 + j];
            float* to = (j & 1) ? db : dD;
            if (to) to[j >> 1] = (float)s;
        }
    }
}

template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_step_kernel(ScanArgs a) {
    const Where w = where(a);
    float h[NS];
    load_state<NS>(a.state0, a, w, h);
    const float x = at_step<T>(a.x, 0, a.x_b, 0, w), z = at_step<T>(a.z, 0, a.z_b, 0, w);
    const float raw = at_step<T>(a.dt, 0, a.dt_b, 0, w) + ((a.bias && w.live) ? a.bias[w.ch] : 0.f);
    const float e = a.softplus ? softplus_f(raw) : raw, u = e * x;
    float p = 0.f;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        if (w.live && n < a.n) {
            const float A2 = a.A[(long long)w.ch * a.n + n] * LOG2E_F;
            h[k] = fmaf(__builtin_amdgcn_exp2f(e * A2), h[k], u * to_f(((const T*)a.B)[w.b * a.B_b + w.g * a.B_g + n]));
            p = fmaf(to_f(((const T*)a.C)[w.b * a.C_b + w.g * a.C_g + n]), h[k], p);
        }
    }
    p = quad_sum(p);
    float y = fmaf((a.D && w.live) ? a.D[w.ch] : 0.f, x, p);
    if (a.z) y *= z * sigmoid_f(z);
    if (w.live && w.q == 0) ((T*)a.y)[(long long)w.b * a.d + w.ch] = from_f<T>(y);
    store_state<NS>(a.state_out, a, w, h);
}

int states_per_lane(int n) { return n <= 4 ? 1 : n <= 8 ? 2 : n <= 16 ? 4 : 8; }
int tile_steps(int n) { return n <= 16 ? 16 : 8; }

template <typename F> int scan_dispatch(int dtype, int n, F f) {
#define JOVA_SCAN_NS(NS)                                                                  \
    {                                                                                     \
        typedef std::integral_constant<int, NS> K;                                        \
        if (dtype == JOVA_F32) return f(float(), K());                                    \
        if (dtype == JOVA_BF16) return f(bf16_t(), K());                                  \
        return f(fp16_t(), K());                                                          \
    }
    switch (states_per_lane(n)) {
        case 1: JOVA_SCAN_NS(1)
        case 2: JOVA_SCAN_NS(2)
        case 4: JOVA_SCAN_NS(4)
        default: JOVA_SCAN_NS(8)
    }
#undef JOVA_SCAN_NS
}

int scan_check(const char* who, int dtype, int64_t steps, int64_t batch, int d, int groups, int n) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype), "%s: unknown dtype %d", who, dtype);
    JOVA_CHECK_ARG(steps >= 0 && batch >= 0 && d >= 1 && groups >= 1 && n >= 1 && d % groups == 0, "%s: bad shape", who);
    if (n > 32 || batch > 65535) {
        jova_set_error("%s: %d states (at most 32), %lld sequences (at most 65535)", who, n, (long long)batch);
        return JOVA_ERR_LIMIT;
    }
    return JOVA_OK;
}

ScanArgs scan_args(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* D, const void* z,
                   const float* bias, int64_t steps, int64_t batch, int d, int groups, int n, const int64_t* st, int softplus,
                   const int32_t* lengths, const float* state0) {
    ScanArgs a = {};
    a.x = x; a.dt = dt; a.A = A; a.B = B; a.C = C; a.D = D; a.z = z; a.bias = bias; a.steps = steps; a.batch = (int)batch;
    a.d = d; a.groups = groups; a.n = n; a.softplus = softplus; a.lengths = lengths; a.state0 = state0;
    a.x_t = st[0]; a.x_b = st[1]; a.dt_t = st[2]; a.dt_b = st[3]; a.z_t = st[4]; a.z_b = st[5];
    a.B_t = st[6]; a.B_b = st[7]; a.B_g = st[8]; a.C_t = st[9]; a.C_b = st[10]; a.C_g = st[11];
    return a;
}

dim3 scan_grid(const ScanArgs& a) {
    const int dg = a.d / a.groups;
    return dim3((unsigned)(a.groups * ((dg + CH - 1) / CH)), (unsigned)a.batch);
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

extern "C" size_t jova_selective_scan_checkpoint_bytes(int64_t steps, int64_t batch, int d, int n_state) {
    if (steps <= 0 || batch <= 0 || d < 1 || n_state < 1 || n_state > 32) return 256;
    const int kt = tile_steps(n_state);
    return (size_t)((steps + kt - 1) / kt) * batch * d * 4 * states_per_lane(n_state) * 4;
}

extern "C" int jova_selective_scan_fwd(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                       const float* D_or_null, const void* z_or_null, const float* dt_bias_or_null, int dtype,
                                       int64_t steps, int64_t batch, int d, int groups, int n_state, const int64_t* strides,
                                       int softplus, const int32_t* lengths_or_null, const float* state0_or_null, void* y,
                                       float* state_out_or_null, void* checkpoints_or_null, void* stream) {
    if (const int rc = scan_check("selective_scan_fwd", dtype, steps, batch, d, groups, n_state)) return rc;
    JOVA_CHECK_ARG(A && strides && (steps * batch == 0 || (x && dt && B && C && y)), "selective_scan_fwd: null pointer");
    if (batch == 0) return JOVA_OK;
    ScanArgs a = scan_args(x, dt, A, B, C, D_or_null, z_or_null, dt_bias_or_null, steps, batch, d, groups, n_state, strides, softplus,
                           lengths_or_null, state0_or_null);
    a.y = y; a.state_out = state_out_or_null; a.ckpt = (float*)checkpoints_or_null;
    return scan_dispatch(dtype, n_state, [&](auto t, auto k) {
        hipLaunchKernelGGL((scan_fwd_kernel<decltype(t), decltype(k)::value>), scan_grid(a), dim3(256), 0, (hipStream_t)stream, a);
        JOVA_CHECK_LAUNCH("selective_scan_fwd");
        return JOVA_OK;
    });
}

extern "C" size_t jova_selective_scan_bwd_workspace_bytes(int64_t steps, int64_t batch, int d, int groups, int n_state) {
    if (steps < 0 || batch <= 0 || d < 1 || groups < 1 || n_state < 1 || n_state > 32) return 256;
    const size_t np = 4 * states_per_lane(n_state), tiles = (d / groups + CH - 1) / CH;
    return align256(tiles * steps * batch * groups * 2 * np * 4) + align256((size_t)batch * d * np * 4) + align256((size_t)batch * d * 8);
}

extern "C" int jova_selective_scan_bwd(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                       const float* D_or_null, const void* z_or_null, const float* dt_bias_or_null, int dtype,
                                       int64_t steps, int64_t batch, int d, int groups, int n_state, const int64_t* strides,
                                       int softplus, const int32_t* lengths_or_null, const void* dy, int64_t dy_t, int64_t dy_b,
                                       const float* dstate_out_or_null, const void* checkpoints, void* dx, void* ddt, void* dz_or_null,
                                       float* dA, void* dB, void* dC, float* dD_or_null, float* dbias_or_null,
                                       float* dstate0_or_null, void* workspace, void* stream) {
    if (const int rc = scan_check("selective_scan_bwd", dtype, steps, batch, d, groups, n_state)) return rc;
    JOVA_CHECK_ARG(A && strides && dA && workspace, "selective_scan_bwd: null pointer");
    JOVA_CHECK_ARG(steps * batch == 0 || (x && dt && B && C && dy && checkpoints && dx && ddt && dB && dC), "selective_scan_bwd: null pointer");
    JOVA_CHECK_ARG(!z_or_null || dz_or_null, "selective_scan_bwd: z without dz");
    ScanArgs a = scan_args(x, dt, A, B, C, D_or_null, z_or_null, dt_bias_or_null, steps, batch, d, groups, n_state, strides, softplus,
                           lengths_or_null, nullptr);
    const int np = 4 * states_per_lane(n_state), tiles = (d / groups + CH - 1) / CH;
    char* ws = (char*)workspace;
    a.part_bc = (float*)ws;
    a.part_a = (float*)(ws + align256((size_t)tiles * steps * batch * groups * 2 * np * 4));
    a.part_d = (float*)((char*)a.part_a + align256((size_t)batch * d * np * 4));
    a.dy = dy; a.dy_t = dy_t; a.dy_b = dy_b; a.dstate_out = dstate_out_or_null; a.ckpt = (float*)checkpoints;
    a.dx = dx; a.ddt = ddt; a.dz = dz_or_null; a.dstate0 = dstate0_or_null;
    const hipStream_t s = (hipStream_t)stream;
    if (batch > 0) {
        const int rc = scan_dispatch(dtype, n_state, [&](auto t, auto k) {
            typedef decltype(t) T;
            hipLaunchKernelGGL((scan_bwd_kernel<T, decltype(k)::value>), scan_grid(a), dim3(256), 0, s, a);
            JOVA_CHECK_LAUNCH("selective_scan_bwd");
            const long long rows = (long long)steps * batch * groups, total = rows * 2 * np;
            if (total) {
                hipLaunchKernelGGL((scan_fold_bc_kernel<T>), dim3((unsigned)(total + 255 < 256ll * 4096 ? (total + 255) / 256 : 4096)), dim3(256), 0,
                                   s, a.part_bc, rows, tiles, np, n_state, (T*)dB, (T*)dC);
                JOVA_CHECK_LAUNCH("selective_scan_bwd (dB, dC)");
            }
            return JOVA_OK;
        });
        if (rc) return rc;
    }
    const long long cols = (long long)d * (np + 2);
    hipLaunchKernelGGL(scan_fold_params_kernel, dim3((unsigned)((cols + 255) / 256)), dim3(256), 0, s, a.part_a, a.part_d, (int)batch, d, np,
                       n_state, dA, dD_or_null, dbias_or_null);
    JOVA_CHECK_LAUNCH("selective_scan_bwd (parameters)");
    return JOVA_OK;
}

extern "C" int jova_selective_scan_step(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                        const float* D_or_null, const void* z_or_null, const float* dt_bias_or_null, int dtype,
                                        int64_t batch, int d, int groups, int n_state, const int64_t* strides, int softplus,
                                        const float* state, float* state_out, void* y, void* stream) {
    if (const int rc = scan_check("selective_scan_step", dtype, 1, batch, d, groups, n_state)) return rc;
    JOVA_CHECK_ARG(A && strides && (batch == 0 || (x && dt && B && C && state && state_out && y)), "selective_scan_step: null pointer");
    if (batch == 0) return JOVA_OK;
    ScanArgs a = scan_args(x, dt, A, B, C, D_or_null, z_or_null, dt_bias_or_null, 1, batch, d, groups, n_state, strides, softplus,
                           nullptr, state);
    a.y = y; a.state_out = state_out;
    return scan_dispatch(dtype, n_state, [&](auto t, auto k) {
        hipLaunchKernelGGL((scan_step_kernel<decltype(t), decltype(k)::value>), scan_grid(a), dim3(256), 0, (hipStream_t)stream, a);
        JOVA_CHECK_LAUNCH("selective_scan_step");
        return JOVA_OK;
    });
}
