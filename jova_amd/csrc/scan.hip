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
constexpr int MAX_CHUNKS = 64, FWD_TARGET = 1024, BWD_TARGET = 512;
template <int NS> struct Tile { static constexpr int KT = NS <= 4 ? 16 : 8; };      // steps between saved states

struct ScanArgs {
    const void *x, *dt, *B, *C, *z, *dy;
    const float *A, *D, *bias, *state0, *dstate_out;
    void *y, *dx, *ddt, *dz;
    float *state_out, *dstate0;
    float* ckpt;                                       // [tiles][batch][d][4 NS]: the state in front of every tile
    float *carry, *esum;                               // [chunks][batch][d][4 NS] and [chunks][batch][d]: carry_in
    float *part_bc, *part_a, *part_d;                  // partial sums of dB | dC, dA, dD | dbias
    const int* lengths;
    long long x_t, x_b, dt_t, dt_b, z_t, z_b, B_t, B_b, B_g, C_t, C_b, C_g, dy_t, dy_b;
    long long steps, chunk;                            // steps of a chunk (blockIdx.z), a multiple of KT
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

// One value per lane: element (t, b, channel) of a [steps, batch, d] tensor, t = tile + 4 j + q.  What is the same for the wave
// stays in scalar registers and moves on with the tiles; the lane's own part is a 32-bit offset that never changes (strides
// are checked on the host: lane_ok).
template <typename T> struct Lane {
    const char* at;                                    // of the tile, batch element b
    long long step4;                                   // bytes of four steps
    unsigned off;                                      // (q * step + channel), bytes
    __device__ __forceinline__ Lane(const void* p, long long s_t, long long s_b, const Where& w, long long t0)
        : at((const char*)p + (t0 * s_t + w.b * s_b) * (long long)sizeof(T)), step4(4 * s_t * (long long)sizeof(T)),
          off((unsigned)(w.q * s_t + w.ch) * (unsigned)sizeof(T)) {}
    __device__ __forceinline__ T load(int j) const { return *(const T*)(at + j * step4 + off); }
    __device__ __forceinline__ void store(int j, float v) const { *(T*)(const_cast<char*>(at) + j * step4 + off) = from_f<T>(v); }
    __device__ __forceinline__ void move(int tiles_j) { at += tiles_j * step4; }
    // values of a tile's steps, those before `rem` (of the sequence) as computed, the others (of the tensor) as zeros
    template <int J> __device__ __forceinline__ void store_tile(const float* v, int rem, int there, int q) const {
        if (rem >= 4 * J) {
#pragma unroll
            for (int j = 0; j < J; ++j) store(j, v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (4 * j + q < there) store(j, 4 * j + q < rem ? v[j] : 0.f);
        }
    }
};
// steps of a tile that are left of `len`
template <int KT> __device__ __forceinline__ int left_of(long long len, long long t0) {
    const long long r = len - t0;
    return r >= KT ? KT : r < 0 ? 0 : (int)r;
}
// a tile's values as stored; steps behind the end are not touched
template <typename T, int J> struct Steps {
    T v[J];
    __device__ __forceinline__ void load(const Lane<T>& l, int rem, int q) {
        if (rem >= 4 * J) {
#pragma unroll
            for (int j = 0; j < J; ++j) v[j] = l.load(j);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j) v[j] = 4 * j + q < rem ? l.load(j) : from_f<T>(0.f);
        }
    }
};

// a tile's rows of B and C -> LDS, fp32, zero behind the sequence and in the padded states
template <typename T, int NS>
struct Rows {
    static constexpr int KT = Tile<NS>::KT, NP = 4 * NS, PER = (2 * KT * NP + 255) / 256;
    T v[PER];
    const char* at[PER];
    long long tile[PER];                               // bytes of a tile
    int t[PER];                                        // step within the tile; KT: nothing to load
    __device__ __forceinline__ Rows(const ScanArgs& a, const Where& w, long long t0, bool with_B) {
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int i = threadIdx.x + 256 * r, n = i % NP;
            const bool isB = i < KT * NP;
            t[r] = (i / NP) % KT;
            const long long s_t = isB ? a.B_t : a.C_t;
            at[r] = (const char*)(isB ? a.B : a.C) +
                    ((t0 + t[r]) * s_t + w.b * (isB ? a.B_b : a.C_b) + w.g * (isB ? a.B_g : a.C_g) + n) * (long long)sizeof(T);
            tile[r] = KT * s_t * (long long)sizeof(T);
            if (i >= 2 * KT * NP || n >= a.n || (isB && !with_B)) t[r] = KT;
        }
    }
    __device__ __forceinline__ void load(int rem) {
#pragma unroll
        for (int r = 0; r < PER; ++r) v[r] = t[r] < rem ? *(const T*)at[r] : from_f<T>(0.f);
    }
    __device__ __forceinline__ void move(int tiles) {
#pragma unroll
        for (int r = 0; r < PER; ++r) at[r] += tiles * tile[r];
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (PER * 256 == 2 * KT * NP || threadIdx.x + 256 * r < 2 * KT * NP) lds[threadIdx.x + 256 * r] = to_f(v[r]);
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
template <int NS> struct alignas(4 * NS) Part { float v[NS]; };
// a lane's NS states in an array [rows][batch][d][4 NS]
template <int NS> __device__ __forceinline__ Part<NS>* part_at(float* p, const ScanArgs& a, const Where& w, long long row) {
    return reinterpret_cast<Part<NS>*>(p) + ((row * a.batch + w.b) * a.d + w.ch) * 4 + w.q;
}
template <int NS> __device__ __forceinline__ void load_A2(const ScanArgs& a, const Where& w, float* A2) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const int n = w.q * NS + k;
        A2[k] = (w.live && n < a.n) ? a.A[(long long)w.ch * a.n + n] * LOG2E_F : 0.f;
    }
}
// The state that enters a chunk: the chunks in front of it (behind it, for the adjoint) are each a product with exp(A sum e)
// and an addition of what they give from zero.
template <int NS> __device__ __forceinline__ void carry_in(const ScanArgs& a, const Where& w, const float* A2, int from, int to, int by, float* h) {
    for (int c = from; c != to; c += by) {
        const Part<NS> p = *part_at<NS>(a.carry, a, w, c);
        const float e = a.esum[((long long)c * a.batch + w.b) * a.d + w.ch];
#pragma unroll
        for (int k = 0; k < NS; ++k) h[k] = fmaf(__builtin_amdgcn_exp2f(e * A2[k]), h[k], p.v[k]);
    }
}
template <typename F> __device__ __forceinline__ void four(F f) {
    f(std::integral_constant<int, 0>());
    f(std::integral_constant<int, 1>());
    f(std::integral_constant<int, 2>());
    f(std::integral_constant<int, 3>());
}
template <typename F> __device__ __forceinline__ void four_back(F f) {
    f(std::integral_constant<int, 3>());
    f(std::integral_constant<int, 2>());
    f(std::integral_constant<int, 1>());
    f(std::integral_constant<int, 0>());
}

// The loops below have no branch between a tile's loads and its stores: options (softplus, the gate) are selects, without z its
// loads read x.

// LOCAL: the chunk's own contribution to the state (from zero) and its sum of e, for carry_in
template <typename T, int NS, bool LOCAL>
__global__ void __launch_bounds__(256)
scan_fwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS, J = KT / 4;
    __shared__ __align__(16) float rows[2][2 * KT * NP];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2, softplus = a.softplus, gate = a.z != nullptr;
    const long long first = (long long)blockIdx.z * a.chunk, last = min(a.steps, first + a.chunk);
    float A2[NS], h[NS], es = 0.f;
    load_A2<NS>(a, w, A2);
    if (LOCAL) {
#pragma unroll
        for (int k = 0; k < NS; ++k) h[k] = 0.f;
    } else {
        load_state<NS>(a.state0, a, w, h);
        carry_in<NS>(a, w, A2, 0, blockIdx.z, 1, h);
    }
    const float Dv = a.D ? a.D[w.ch] : 0.f, bias = a.bias ? a.bias[w.ch] : 0.f;
    Lane<T> lx(a.x, a.x_t, a.x_b, w, first), ldt(a.dt, a.dt_t, a.dt_b, w, first);
    Lane<T> lz(gate ? a.z : a.x, gate ? a.z_t : a.x_t, gate ? a.z_b : a.x_b, w, first), ly(a.y, (long long)a.batch * a.d, a.d, w, first);
    Rows<T, NS> rn(a, w, first, true);
    Steps<T, J> xn, dn, zn;
    int rem = left_of<KT>(w.len, first);
    auto fetch = [&]() {
        rn.load(rem);
        xn.load(lx, rem, w.q);
        dn.load(ldt, rem, w.q);
        if (!LOCAL) zn.load(lz, rem, w.q);
    };
    fetch();
    rn.put(rows[0]);
    __syncthreads();
    int cur = 0;
    for (long long t0 = first; t0 < last; t0 += KT, cur ^= 1) {
        float x[J], e[J], z[J], y[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = to_f(xn.v[j]);
            const float raw = to_f(dn.v[j]) + bias, sp = softplus_f(raw);
            e[j] = 4 * j + w.q < rem ? (softplus ? sp : raw) : 0.f;
            if (!LOCAL) z[j] = to_f(zn.v[j]);
        }
        const int now = rem;
        const bool more = t0 + KT < last;
        if (more) {
            rn.move(1);
            lx.move(J);
            ldt.move(J);
            lz.move(J);
            rem = left_of<KT>(w.len, t0 + KT);
            fetch();
        }
        if (!LOCAL && a.ckpt && w.live) {
            Part<NS> p;
#pragma unroll
            for (int k = 0; k < NS; ++k) p.v[k] = h[k];
            *part_at<NS>(a.ckpt, a, w, t0 / KT) = p;
        }
        const float* lds = rows[cur] + w.q * NS;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float p[4];
            const float u = e[j] * x[j];
            if (LOCAL) es += e[j];
            four([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const float ei = quad_bcast<i>(e[j]), ui = quad_bcast<i>(u);
                const float *Bt = lds + (4 * j + i) * NP, *Ct = Bt + KT * NP;
                p[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    h[k] = fmaf(__builtin_amdgcn_exp2f(ei * A2[k]), h[k], ui * Bt[k]);
                    if (!LOCAL) p[i] = fmaf(Ct[k], h[k], p[i]);
                }
            });
            if (!LOCAL) {
                const float v = fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1));
                y[j] = gate ? v * (z[j] * sigmoid_f(z[j])) : v;
            }
        }
        if (!LOCAL) {
            if (w.live) ly.template store_tile<J>(y, now, left_of<KT>(a.steps, t0), w.q);
            ly.move(J);
        }
        if (more) rn.put(rows[cur ^ 1]);
        __syncthreads();
    }
    if (LOCAL) {
        es = quad_sum(es);
        if (!w.live) return;
        Part<NS> p;
#pragma unroll
        for (int k = 0; k < NS; ++k) p.v[k] = h[k];
        *part_at<NS>(a.carry, a, w, blockIdx.z) = p;
        if (w.q == 0) a.esum[((long long)blockIdx.z * a.batch + w.b) * a.d + w.ch] = es;
    } else if (blockIdx.z + 1 == gridDim.z) {
        store_state<NS>(a.state_out, a, w, h);
    }
}

// The adjoint that a chunk hands to the one in front of it, from zero: q <- exp(e A) (q + C g), steps descending
template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_adjoint_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS, J = KT / 4;
    __shared__ __align__(16) float rows[2][2 * KT * NP];
    const Where w = where(a);
    const bool softplus = a.softplus, gate = a.z != nullptr;
    const int chunk = blockIdx.z + 1;                  // nothing is in front of chunk 0
    const long long first = (long long)chunk * a.chunk, last = min(a.steps, first + a.chunk), top = first + ((last - first - 1) / KT) * KT;
    float A2[NS], q[NS], es = 0.f;
    load_A2<NS>(a, w, A2);
#pragma unroll
    for (int k = 0; k < NS; ++k) q[k] = 0.f;
    const float bias = a.bias ? a.bias[w.ch] : 0.f;
    Lane<T> ldt(a.dt, a.dt_t, a.dt_b, w, top), ldy(a.dy, a.dy_t, a.dy_b, w, top);
    Lane<T> lz(gate ? a.z : a.dy, gate ? a.z_t : a.dy_t, gate ? a.z_b : a.dy_b, w, top);
    Rows<T, NS> rn(a, w, top, false);
    Steps<T, J> dn, zn, gn;
    int rem = left_of<KT>(w.len, top);
    auto fetch = [&]() {
        rn.load(rem);
        dn.load(ldt, rem, w.q);
        gn.load(ldy, rem, w.q);
        zn.load(lz, rem, w.q);
    };
    fetch();
    rn.put(rows[0]);
    __syncthreads();
    int cur = 0;
    for (long long t0 = top; t0 >= first; t0 -= KT, cur ^= 1) {
        float e[J], g[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float raw = to_f(dn.v[j]) + bias, sp = softplus_f(raw), z = to_f(zn.v[j]), dy = to_f(gn.v[j]);
            e[j] = 4 * j + w.q < rem ? (softplus ? sp : raw) : 0.f;
            g[j] = gate ? dy * (z * sigmoid_f(z)) : dy;
            es += e[j];
        }
        const bool more = t0 > first;
        if (more) {
            rn.move(-1);
            ldt.move(-J);
            ldy.move(-J);
            lz.move(-J);
            rem = left_of<KT>(w.len, t0 - KT);
            fetch();
        }
        const float* lds = rows[cur] + KT * NP + w.q * NS;
#pragma unroll
        for (int j = J - 1; j >= 0; --j)
            four_back([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const float ei = quad_bcast<i>(e[j]), gi = quad_bcast<i>(g[j]);
                const float* Ct = lds + (4 * j + i) * NP;
#pragma unroll
                for (int k = 0; k < NS; ++k) q[k] = fmaf(Ct[k], gi, q[k]) * __builtin_amdgcn_exp2f(ei * A2[k]);
            });
        if (more) rn.put(rows[cur ^ 1]);
        __syncthreads();
    }
    es = quad_sum(es);
    if (!w.live) return;
    Part<NS> p;
#pragma unroll
    for (int k = 0; k < NS; ++k) p.v[k] = q[k];
    *part_at<NS>(a.carry, a, w, chunk) = p;
    if (w.q == 0) a.esum[((long long)chunk * a.batch + w.b) * a.d + w.ch] = es;
}

__device__ __forceinline__ unsigned bits(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float swap32_sum(float a, float b) {        // lanes 0-31: a over both halves, lanes 32-63: b
    const auto r = __builtin_amdgcn_permlane32_swap(bits(a), bits(b), false, false);
    const unsigned lo = r[0], hi = r[1];               // (bit_cast of a vector's element reads element 0)
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float swap16_sum(float a, float b) {        // even rows of 16 lanes: a over a pair of rows, odd rows: b
    const auto r = __builtin_amdgcn_permlane16_swap(bits(a), bits(b), false, false);
    const unsigned lo = r[0], hi = r[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
// Sums over the wave's 16 channels of v[2][4][NS] (dB | dC, step, state): halved four times, every halving one exchange of
// lanes and one addition a pair.  Lane l is left with kind l5, step (l4, l3) and the max(NS / 2, 1) states from l2 NS / 2.
template <int NS> __device__ __forceinline__ void channel_sums(float* v, int lane) {
#pragma unroll
    for (int i = 0; i < 4 * NS; ++i) v[i] = swap32_sum(v[i], v[i + 4 * NS]);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) v[i] = swap16_sum(v[i], v[i + 2 * NS]);
    const bool l3 = lane & 8, l2 = lane & 4;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const float lo = v[i] + dpp<0x128>(v[i]), hi = v[i + NS] + dpp<0x128>(v[i + NS]);        // row_ror:8 = the lane with bit 3 flipped
        v[i] = l3 ? hi : lo;
    }
    if (NS == 1) {
        const float lo = v[0] + dpp<0x104>(v[0]), hi = v[0] + dpp<0x114>(v[0]);                  // row_shl:4, row_shr:4
        v[0] = l2 ? hi : lo;
    } else {
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
            const float lo = v[i] + dpp<0x104>(v[i]), hi = v[i + NS / 2] + dpp<0x114>(v[i + NS / 2]);
            v[i] = l2 ? hi : lo;
        }
    }
}

template <typename T, int NS>
__global__ void __launch_bounds__(256, 2)
scan_bwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS, J = KT / 4, HALF = NS > 1 ? NS / 2 : 1;
    __shared__ __align__(16) float rows[2 * KT * NP];
    __shared__ __align__(16) float red[WAVES][KT][2][NP];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2, softplus = a.softplus, gate = a.z != nullptr;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long first = (long long)blockIdx.z * a.chunk, last = min(a.steps, first + a.chunk);
    const long long top = last > first ? first + ((last - first - 1) / KT) * KT : first - KT;
    float A2[NS], q[NS], dA[NS], dD = 0.f, db = 0.f;
    load_A2<NS>(a, w, A2);
    load_state<NS>(a.dstate_out, a, w, q);
    carry_in<NS>(a, w, A2, (int)gridDim.z - 1, (int)blockIdx.z, -1, q);
#pragma unroll
    for (int k = 0; k < NS; ++k) dA[k] = 0.f;
    const float Dv = a.D ? a.D[w.ch] : 0.f, bias = a.bias ? a.bias[w.ch] : 0.f;
    const long long o_t = (long long)a.batch * a.d;
    Lane<T> lx(a.x, a.x_t, a.x_b, w, top), ldt(a.dt, a.dt_t, a.dt_b, w, top), ldy(a.dy, a.dy_t, a.dy_b, w, top);
    Lane<T> lz(gate ? a.z : a.x, gate ? a.z_t : a.x_t, gate ? a.z_b : a.x_b, w, top);
    Lane<T> odx(a.dx, o_t, a.d, w, top), oddt(a.ddt, o_t, a.d, w, top), odz(a.dz, o_t, a.d, w, top);
    Rows<T, NS> rn(a, w, top, true);
    for (long long t0 = top; t0 >= first; t0 -= KT) {
        const int rem = left_of<KT>(w.len, t0), there = left_of<KT>(a.steps, t0);
        Steps<T, J> xn, dn, zn, gn;
        rn.load(rem);
        const Part<NS> h0 = *part_at<NS>(a.ckpt, a, w, t0 / KT);
        xn.load(lx, rem, w.q);
        dn.load(ldt, rem, w.q);
        gn.load(ldy, rem, w.q);
        zn.load(lz, rem, w.q);
        float x[J], e[J], raw[J], g[J], hs[KT][NS], as[KT][NS];
        rn.put(rows);
        __syncthreads();
        const float* lds = rows + w.q * NS;
        // the tile's states once more, and the output in front of the gate
        float dz[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = w.live ? to_f(xn.v[j]) : 0.f;
            raw[j] = to_f(dn.v[j]) + bias;
            const float sp = softplus_f(raw[j]);
            e[j] = 4 * j + w.q < rem ? (softplus ? sp : raw[j]) : 0.f;
            const float dy = w.live ? to_f(gn.v[j]) : 0.f, u = e[j] * x[j];
            float p[4];
            four([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = 4 * j + i;
                const float ei = quad_bcast<i>(e[j]), ui = quad_bcast<i>(u);
                const float *Bt = lds + t * NP, *Ct = Bt + KT * NP;
                p[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    as[t][k] = __builtin_amdgcn_exp2f(ei * A2[k]);
                    hs[t][k] = fmaf(as[t][k], t > 0 ? hs[t > 0 ? t - 1 : 0][k] : h0.v[k], ui * Bt[k]);
                    p[i] = fmaf(Ct[k], hs[t][k], p[i]);
                }
            });
            const float pre = fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1)), z = to_f(zn.v[j]), sg = sigmoid_f(z);
            g[j] = gate ? dy * (z * sg) : dy;
            dz[j] = dy * pre * (sg * (1.f + z * (1.f - sg)));
            dD = fmaf(g[j], x[j], dD);
        }
        if (gate && w.live) odz.template store_tile<J>(dz, rem, there, w.q);
        float dAt[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) dAt[k] = 0.f;
#pragma unroll
        for (int j = J - 1; j >= 0; --j) {
            float pb[4], pf[4], v[8 * NS];
            const float u = e[j] * x[j];
            four_back([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = 4 * j + i;
                const float gi = quad_bcast<i>(g[j]), ui = quad_bcast<i>(u), ei = quad_bcast<i>(e[j]);
                const float *Bt = lds + t * NP, *Ct = Bt + KT * NP;
                pb[i] = pf[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    q[k] = fmaf(Ct[k], gi, q[k]);
                    pb[i] = fmaf(q[k], Bt[k], pb[i]);
                    v[i * NS + k] = q[k] * ui;
                    v[(4 + i) * NS + k] = gi * hs[t][k];
                    q[k] *= as[t][k];
                    const float f = q[k] * (t > 0 ? hs[t > 0 ? t - 1 : 0][k] : h0.v[k]);
                    dAt[k] = fmaf(f, ei, dAt[k]);
                    pf[i] = fmaf(f, A2[k], pf[i]);
                }
            });
            channel_sums<NS>(v, lane);
            {
                float* to = &red[wave][4 * j + ((lane >> 3) & 3)][lane >> 5][w.q * NS + (NS > 1 && (lane & 4) ? NS / 2 : 0)];
#pragma unroll
                for (int k = 0; k < HALF; ++k) to[k] = v[k];       // (NS = 1: both lanes write the same sum)
            }
            const float qb = quad_scatter_sum(pb, b0, b1), fa = quad_scatter_sum(pf, b0, b1) * LN2_F;
            const float de = fmaf(qb, x[j], fa), sl = sigmoid_f(raw[j]);
            raw[j] = 4 * j + w.q < rem ? (softplus ? de * sl : de) : 0.f;              // now the gradient of dt
            db += raw[j];
            x[j] = fmaf(g[j], Dv, qb * e[j]);                                          // now the gradient of x
        }
        if (w.live) {
            odx.template store_tile<J>(x, rem, there, w.q);
            oddt.template store_tile<J>(raw, rem, there, w.q);
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) dA[k] += dAt[k];
        __syncthreads();
        for (int i = threadIdx.x; i < KT * 2 * NP; i += 256) {
            const int t = i / (2 * NP);
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) s += (&red[v][0][0][0])[i];
            if (t < there)
                a.part_bc[((((long long)w.tile * a.steps + t0 + t) * a.batch + w.b) * a.groups + w.g) * 2 * NP + i % (2 * NP)] = s;
        }
        rn.move(-1);
        lx.move(-J);
        ldt.move(-J);
        ldy.move(-J);
        lz.move(-J);
        odx.move(-J);
        oddt.move(-J);
        odz.move(-J);
    }
    if (blockIdx.z == 0) store_state<NS>(a.dstate0, a, w, q);
    dD = quad_sum(dD);
    db = quad_sum(db);
    if (w.live) {
        const long long row = ((long long)blockIdx.z * a.batch + w.b) * a.d + w.ch;
        Part<NS> p;
#pragma unroll
        for (int k = 0; k < NS; ++k) p.v[k] = dA[k];
        reinterpret_cast<Part<NS>*>(a.part_a)[row * 4 + w.q] = p;
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

template <typename T> __device__ __forceinline__ float of_token(const void* p, long long s_b, const Where& w) {
    return p ? to_f(((const T*)p)[w.b * s_b + w.ch]) : 0.f;
}
template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_step_kernel(ScanArgs a) {
    const Where w = where(a);
    float h[NS];
    load_state<NS>(a.state0, a, w, h);
    const float x = of_token<T>(a.x, a.x_b, w), z = of_token<T>(a.z, a.z_b, w);
    const float raw = of_token<T>(a.dt, a.dt_b, w) + (a.bias ? a.bias[w.ch] : 0.f);
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

int channel_tiles(int d, int groups) { return groups * ((d / groups + CH - 1) / CH); }

// Chunks of the time axis: enough workgroups to fill the card, few enough that the extra pass over the chunks pays.
struct Plan { int chunks; long long chunk; };
Plan scan_plan(int64_t steps, int64_t batch, int d, int groups, int n, int target, int least) {
    const long long kt = tile_steps(n), wgs = (long long)channel_tiles(d, groups) * batch;
    Plan p = {1, (steps + kt - 1) / kt * kt};
    long long c = target / (wgs > 0 ? wgs : 1);
    if (c > steps / least) c = steps / least;
    if (c > MAX_CHUNKS) c = MAX_CHUNKS;
    if (c > 1) {
        p.chunk = ((steps + c - 1) / c + kt - 1) / kt * kt;
        p.chunks = (int)((steps + p.chunk - 1) / p.chunk);
    }
    if (p.chunk < kt) p.chunk = kt;
    return p;
}
Plan fwd_plan(int64_t steps, int64_t batch, int d, int groups, int n) { return scan_plan(steps, batch, d, groups, n, FWD_TARGET, 128); }
Plan bwd_plan(int64_t steps, int64_t batch, int d, int groups, int n) { return scan_plan(steps, batch, d, groups, n, BWD_TARGET, 128); }

dim3 scan_grid(const ScanArgs& a, int z = 1) { return dim3((unsigned)channel_tiles(a.d, a.groups), (unsigned)a.batch, (unsigned)z); }

// Lane's 32-bit offsets: 3 steps and a channel, in bytes
bool lane_ok(const ScanArgs& a) {
    const long long lim = (1ll << 29);
    return 3 * a.x_t + a.d < lim && 3 * a.dt_t + a.d < lim && 3 * a.z_t + a.d < lim && 3 * a.dy_t + a.d < lim &&
           3 * (long long)a.batch * a.d + a.d < lim && a.x_t >= 0 && a.dt_t >= 0 && a.z_t >= 0 && a.dy_t >= 0;
}
#define JOVA_SCAN_LANES(who)                                                                    \
    if (!lane_ok(a)) {                                                                          \
        jova_set_error(who ": a step of more than 2^29 / 3 elements");                          \
        return JOVA_ERR_LIMIT;                                                                  \
    }

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

extern "C" size_t jova_selective_scan_checkpoint_bytes(int64_t steps, int64_t batch, int d, int n_state) {
    if (steps <= 0 || batch <= 0 || d < 1 || n_state < 1 || n_state > 32) return 256;
    const int kt = tile_steps(n_state);
    return (size_t)((steps + kt - 1) / kt) * batch * d * 4 * states_per_lane(n_state) * 4;
}

extern "C" size_t jova_selective_scan_fwd_workspace_bytes(int64_t steps, int64_t batch, int d, int groups, int n_state) {
    if (steps <= 0 || batch <= 0 || d < 1 || groups < 1 || n_state < 1 || n_state > 32) return 256;
    const size_t rows = (size_t)fwd_plan(steps, batch, d, groups, n_state).chunks * batch * d;
    return align256(rows * 4 * states_per_lane(n_state) * 4) + align256(rows * 4);
}

extern "C" int jova_selective_scan_fwd(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                       const float* D_or_null, const void* z_or_null, const float* dt_bias_or_null, int dtype,
                                       int64_t steps, int64_t batch, int d, int groups, int n_state, const int64_t* strides,
                                       int softplus, const int32_t* lengths_or_null, const float* state0_or_null, void* y,
                                       float* state_out_or_null, void* checkpoints_or_null, void* workspace, void* stream) {
    if (const int rc = scan_check("selective_scan_fwd", dtype, steps, batch, d, groups, n_state)) return rc;
    JOVA_CHECK_ARG(A && strides && workspace && (steps * batch == 0 || (x && dt && B && C && y)), "selective_scan_fwd: null pointer");
    if (batch == 0) return JOVA_OK;
    ScanArgs a = scan_args(x, dt, A, B, C, D_or_null, z_or_null, dt_bias_or_null, steps, batch, d, groups, n_state, strides, softplus,
                           lengths_or_null, state0_or_null);
    JOVA_SCAN_LANES("selective_scan_fwd")
    const Plan p = fwd_plan(steps, batch, d, groups, n_state);
    a.y = y; a.state_out = state_out_or_null; a.ckpt = (float*)checkpoints_or_null; a.chunk = p.chunk;
    a.carry = (float*)workspace;
    a.esum = (float*)((char*)workspace + align256((size_t)p.chunks * batch * d * 4 * states_per_lane(n_state) * 4));
    const hipStream_t s = (hipStream_t)stream;
    return scan_dispatch(dtype, n_state, [&](auto t, auto k) {
        typedef decltype(t) T;
        constexpr int NS = decltype(k)::value;
        if (p.chunks > 1) {
            hipLaunchKernelGGL((scan_fwd_kernel<T, NS, true>), scan_grid(a, p.chunks - 1), dim3(256), 0, s, a);
            JOVA_CHECK_LAUNCH("selective_scan_fwd (chunks)");
        }
        hipLaunchKernelGGL((scan_fwd_kernel<T, NS, false>), scan_grid(a, p.chunks), dim3(256), 0, s, a);
        JOVA_CHECK_LAUNCH("selective_scan_fwd");
        return JOVA_OK;
    });
}

namespace {
struct BwdSpace { size_t bc, a, d, carry, esum, all; };
BwdSpace bwd_space(int64_t steps, int64_t batch, int d, int groups, int n, int chunks) {
    const size_t np = 4 * states_per_lane(n), rows = (size_t)chunks * batch * d, tiles = (d / groups + CH - 1) / CH;
    BwdSpace s;
    s.bc = 0;
    s.a = s.bc + align256(tiles * steps * batch * groups * 2 * np * 4);
    s.d = s.a + align256(rows * np * 4);
    s.carry = s.d + align256(rows * 8);
    s.esum = s.carry + align256(rows * np * 4);
    s.all = s.esum + align256(rows * 4);
    return s;
}
}  // namespace

extern "C" size_t jova_selective_scan_bwd_workspace_bytes(int64_t steps, int64_t batch, int d, int groups, int n_state) {
    if (steps < 0 || batch <= 0 || d < 1 || groups < 1 || n_state < 1 || n_state > 32) return 256;
    return bwd_space(steps, batch, d, groups, n_state, bwd_plan(steps, batch, d, groups, n_state).chunks).all;
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
    a.dy = dy; a.dy_t = dy_t; a.dy_b = dy_b; a.dstate_out = dstate_out_or_null; a.ckpt = (float*)checkpoints;
    JOVA_SCAN_LANES("selective_scan_bwd")
    const int np = 4 * states_per_lane(n_state), tiles = (d / groups + CH - 1) / CH;
    const Plan p = bwd_plan(steps, batch, d, groups, n_state);
    const BwdSpace sp = bwd_space(steps, batch, d, groups, n_state, p.chunks);
    char* ws = (char*)workspace;
    a.part_bc = (float*)(ws + sp.bc); a.part_a = (float*)(ws + sp.a); a.part_d = (float*)(ws + sp.d);
    a.carry = (float*)(ws + sp.carry); a.esum = (float*)(ws + sp.esum); a.chunk = p.chunk;
    a.dx = dx; a.ddt = ddt; a.dz = dz_or_null; a.dstate0 = dstate0_or_null;
    const hipStream_t s = (hipStream_t)stream;
    if (batch > 0) {
        const int rc = scan_dispatch(dtype, n_state, [&](auto t, auto k) {
            typedef decltype(t) T;
            constexpr int NS = decltype(k)::value;
            if (p.chunks > 1) {
                hipLaunchKernelGGL((scan_adjoint_kernel<T, NS>), scan_grid(a, p.chunks - 1), dim3(256), 0, s, a);
                JOVA_CHECK_LAUNCH("selective_scan_bwd (chunks)");
            }
            hipLaunchKernelGGL((scan_bwd_kernel<T, NS>), scan_grid(a, p.chunks), dim3(256), 0, s, a);
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
    hipLaunchKernelGGL(scan_fold_params_kernel, dim3((unsigned)((cols + 255) / 256)), dim3(256), 0, s, a.part_a, a.part_d,
                       (int)(batch * p.chunks), d, np, n_state, dA, dD_or_null, dbias_or_null);
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
