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
// The states of a step live in registers and in nothing else; the backward pass starts every 8 steps from a saved state (8 bytes per
// element of x at 16 states) and computes the states between once more.
//
// Bound by the vector ALUs, not by memory: per element and state the forward pass has exp (2 issue slots), e A, u B and two
// multiply-adds, the backward pass about 17 operations, against 8 and 22 bytes per element with 16 states in 16 bits.  Packed fp32
// operations are not used.  B and C come in through LDS, 16 (8) steps at once, two sides, the next tile's loads in flight meanwhile.
// 2048 x 8 x 2048, 16 states, bf16: 772 us a call; chunk states 98 (vector ALUs busy 92 %), forward 165 (90 %), chunk adjoints 83 (93 %),
// backward 398 (86 %), folds 17.  16384 x 1 x 4096: 500 us a call, chunk states 214 (96 %) and forward 285 (97 %).
// 232 x 128 x 512 ragged fp32: 204 us a call; forward 60, backward 135, folds 12 (vector ALUs busy 80
// and 77 % of the time that the CUs have work, which is about 70 % of the kernels': lengths differ, no chunks).
// (Kernels: the fastest of 60 in a trace, whose sums agree with the calls; a trace of 10 ends before the clock has settled.)
#include "seq.h"

#include <type_traits>

namespace {

constexpr int WAVES = 4, CH = 16 * WAVES;              // channels of a workgroup
// Workgroups to aim at when the time axis is cut (scan_plan).  Cutting costs a second pass over all chunks but one, too few
// workgroups leave the SIMDs with one or two waves.  Forward target 256, 512, 768, 1024, 2048, 4096: 16384 x 1 x 4096 takes 978,
// 616, 561, 534, 500, 514 us, 2048 x 8 x 2048 with its backward pass 798, 823, 783, 787, 783, 804; backward target 512, 768, 1536: 880, 783, 791
// (three waves a SIMD are all its registers allow).
constexpr int MAX_CHUNKS = 64, FWD_TARGET = 2048, BWD_TARGET = 768;
// Steps of a chunk at least: with 64, 232 x 128 x 512 (1024 workgroups uncut) would be cut too: 241 against 209 us; 256: no difference.
// All three constants were swept on the shapes named here.  Few workgroups (one sequence of few channels) run a chunk's 128 steps
// in series, in up to four passes: a shorter bound for them was not measured.
constexpr int LEAST_CHUNK = 128;
// Steps of a tile: the forward passes take 16 (loads, address arithmetic and the barrier are shared by more steps), the backward pass
// 8, whose states fit the registers of three waves a SIMD; states are saved every 8 steps.  (16 and two waves: 565 against
// 447 us on 2048 x 8 x 2048; 32 states need twice the registers a step, so 8 in all passes.)
template <int NS> struct Tile { static constexpr int KT = NS <= 4 ? 16 : 8, BACK = 8; };

struct ScanArgs {
    const void *x, *dt, *B, *C, *z, *dy;
    const float *A, *D, *bias, *state0, *dstate_out;
    void *y, *dx, *ddt, *dz;
    float *state_out, *dstate0;
    float* ckpt;                                       // [tiles][batch][d][4 NS]: the state in front of every tile
    float *carry, *esum;                               // [chunks or pieces][batch][d][4 NS] and [..][batch][d]: carry_in
    float *part_bc, *part_a, *part_d;                  // partial sums of dB | dC, dA, dD | dbias
    const int* lengths;
    long long x_t, x_b, dt_t, dt_b, z_t, z_b, B_t, B_b, B_g, C_t, C_b, C_g, dy_t, dy_b;
    int steps, chunk;                                  // steps of a chunk (blockIdx.z), a multiple of KT
    int piece, pieces;                                 // of the adjoint pass: steps of a piece of a chunk, pieces of a chunk
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
    int len;
};
// Sequences of a ragged batch start longest first (up to 256 of them: every workgroup ranks the lengths itself), so that a long one
// does not begin when the others end (232 x 128 x 512 ragged, forward and backward: 263 -> 211 us together with skipping the
// tiles behind the ends).
__device__ __forceinline__ int sequence_of(const ScanArgs& a, int slot) {
    if (!a.lengths || a.batch > 256) return slot;
    __shared__ int len[256], chosen;
    const int t = threadIdx.x, mine = t < a.batch ? a.lengths[t] : 0;
    len[t] = mine;
    __syncthreads();
    int rank = 0;
    for (int k = 0; k < a.batch; ++k) rank += len[k] > mine || (len[k] == mine && k < t);
    if (t < a.batch && rank == slot) chosen = t;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(chosen);
}
__device__ __forceinline__ Where where(const ScanArgs& a) {
    Where w;
    const int dg = a.d / a.groups, tiles = (dg + CH - 1) / CH;
    w.g = blockIdx.x / tiles;
    w.tile = blockIdx.x % tiles;
    w.b = sequence_of(a, blockIdx.y);
    w.q = threadIdx.x & 3;
    const int c = w.tile * CH + (threadIdx.x >> 2);
    w.live = c < dg;
    w.ch = w.g * dg + (w.live ? c : 0);
    w.len = a.lengths ? min(max(a.lengths[w.b], 0), a.steps) : a.steps;
    return w;
}

// One value per lane: element (t, b, channel) of a [steps, batch, d] tensor, t = tile + 4 j + q.  What is the same for the wave
// stays in scalar registers and moves on with the tiles; the lane's own part is a 32-bit offset that never changes (strides
// are checked on the host: lane_ok).
template <typename T> struct Lane {
    const char* at;                                    // of the tile, batch element b
    unsigned step4;                                    // bytes of four steps
    unsigned off;                                      // (q * step + channel), bytes
    __device__ __forceinline__ Lane(const void* p, long long s_t, long long s_b, const Where& w, int t0)
        : at((const char*)p + (t0 * s_t + w.b * s_b) * (long long)sizeof(T)), step4(4u * (unsigned)s_t * (unsigned)sizeof(T)),
          off((unsigned)(w.q * s_t + w.ch) * (unsigned)sizeof(T)) {}
    __device__ __forceinline__ T load(int j) const { return *(const T*)(at + j * step4 + off); }
    __device__ __forceinline__ void store(int j, float v) const { *(T*)(const_cast<char*>(at) + j * step4 + off) = from_f<T>(v); }
    __device__ __forceinline__ void move(int j) { at += (long long)step4 * j; }
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
template <int KT> __device__ __forceinline__ int left_of(int len, int t0) { return min(max(len - t0, 0), KT); }
// values of steps behind the sequence's end -> 0
template <int J> __device__ __forceinline__ void cut_steps(float* v, int rem, int q) {
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = 4 * j + q < rem ? v[j] : 0.f;
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
template <typename T, int NS, int KT>
struct Rows {
    static constexpr int NP = 4 * NS, PER = (2 * KT * NP + 255) / 256;
    T v[PER];
    const char* at[PER];
    long long tile[PER];                               // bytes of a tile
    int t[PER];                                        // step within the tile; KT: nothing to load
    __device__ __forceinline__ Rows(const ScanArgs& a, const Where& w, int t0, bool with_B) {
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
        for (int k = 0; k < NS; ++k)                   // (nothing stays nothing, also where a growing state's factor overflows)
            h[k] = h[k] == 0.f ? p.v[k] : fmaf(__builtin_amdgcn_exp2f(e * A2[k]), h[k], p.v[k]);
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

// The loops below have no branch between a tile's loads and its stores: options (softplus, the gate) are selects (pick keeps the
// compiler from making branches of them), without z its loads read x.
#define pick(c) __builtin_unpredictable(c)

// LOCAL: the chunk's own contribution to the state (from zero) and its sum of e, for carry_in.  In the main pass y's sum over n is
// the lane's NS terms, then one exchange for four steps (quad_scatter_sum) that leaves every lane the step it stores.
template <typename T, int NS, bool LOCAL>
__global__ void __launch_bounds__(256)
scan_fwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS, J = KT / 4;
    __shared__ __align__(16) float rows[2][2 * KT * NP];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2, softplus = a.softplus, gate = a.z != nullptr;
    const int first = blockIdx.z * a.chunk, last = min(a.steps, first + a.chunk), end = min(last, max(first, w.len));
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
    Rows<T, NS, KT> rn(a, w, first, true);
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
    Part<NS>* ck = (!LOCAL && a.ckpt && w.live) ? part_at<NS>(a.ckpt, a, w, first / Tile<NS>::BACK) : nullptr;
    const long long ck_tile = (long long)a.batch * a.d * 4;
    int cur = 0;
    int t0 = first;
    for (; t0 < end; t0 += KT, cur ^= 1) {
        float x[J], e[J], gz[J], y[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = to_f(xn.v[j]);
            const float raw = to_f(dn.v[j]) + bias, sp = softplus_f(raw);
            e[j] = pick(softplus) ? sp : raw;
            if (!LOCAL) {
                const float z = to_f(zn.v[j]), zs = z * sigmoid_f(z);
                gz[j] = pick(gate) ? zs : 1.f;
            }
        }
        if (rem < KT) cut_steps<J>(e, rem, w.q);
        const int now = rem;
        const bool more = t0 + KT < end;
        if (more) {
            rn.move(1);
            lx.move(J);
            ldt.move(J);
            lz.move(J);
            rem = left_of<KT>(w.len, t0 + KT);
            fetch();
        }
        const float* lds = rows[cur] + w.q * NS;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float p[4];
            const float u = e[j] * x[j];
            if (LOCAL) es += e[j];
            if (!LOCAL && ck && (4 * j) % Tile<NS>::BACK == 0 && t0 + 4 * j < a.steps) {
                Part<NS> c;
#pragma unroll
                for (int k = 0; k < NS; ++k) c.v[k] = h[k];
                *ck = c;
                ck += ck_tile;
            }
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
            if (!LOCAL) y[j] = fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1)) * gz[j];
        }
        if (!LOCAL) {
            if (w.live) ly.template store_tile<J>(y, now, left_of<KT>(a.steps, t0), w.q);
            ly.move(J);
        }
        if (more) rn.put(rows[cur ^ 1]);
        __syncthreads();
    }
    if (!LOCAL && w.live) {                            // tiles behind the sequence's end
        const float none[J] = {};
        for (; t0 < last; t0 += KT, ly.move(J)) ly.template store_tile<J>(none, 0, left_of<KT>(a.steps, t0), w.q);
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

// The adjoint that a piece of a chunk hands to what is in front of it, from zero: q <- exp(e A) (q + C g), steps descending.  Its
// registers allow more waves than the backward pass, whose chunks are cut into pieces for it (bwd_plan).
template <typename T, int NS>
__global__ void __launch_bounds__(256)
scan_adjoint_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::KT, NP = 4 * NS, J = KT / 4;
    __shared__ __align__(16) float rows[2][2 * KT * NP];
    const Where w = where(a);
    const bool softplus = a.softplus, gate = a.z != nullptr;
    const int chunk = 1 + blockIdx.z / a.pieces, row = blockIdx.z + a.pieces;          // nothing is in front of chunk 0
    const int first = chunk * a.chunk + blockIdx.z % a.pieces * a.piece;
    const int end = min(min(a.steps, min(first + a.piece, (chunk + 1) * a.chunk)), max(first, w.len));
    const int top = end > first ? first + ((end - first - 1) / KT) * KT : first - KT;
    float A2[NS], q[NS], es = 0.f;
    load_A2<NS>(a, w, A2);
#pragma unroll
    for (int k = 0; k < NS; ++k) q[k] = 0.f;
    const float bias = a.bias ? a.bias[w.ch] : 0.f;
    Lane<T> ldt(a.dt, a.dt_t, a.dt_b, w, top), ldy(a.dy, a.dy_t, a.dy_b, w, top);
    Lane<T> lz(gate ? a.z : a.dy, gate ? a.z_t : a.dy_t, gate ? a.z_b : a.dy_b, w, top);
    Rows<T, NS, KT> rn(a, w, top, false);
    Steps<T, J> dn, zn, gn;
    int rem = left_of<KT>(w.len, top);
    auto fetch = [&]() {
        rn.load(rem);
        dn.load(ldt, rem, w.q);
        gn.load(ldy, rem, w.q);
        zn.load(lz, rem, w.q);
    };
    if (top >= first) {
        fetch();
        rn.put(rows[0]);
    }
    __syncthreads();
    int cur = 0;
    for (int t0 = top; t0 >= first; t0 -= KT, cur ^= 1) {
        float e[J], g[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float raw = to_f(dn.v[j]) + bias, sp = softplus_f(raw), z = to_f(zn.v[j]), dy = to_f(gn.v[j]);
            const float zs = z * sigmoid_f(z);
            e[j] = pick(softplus) ? sp : raw;
            g[j] = dy * (pick(gate) ? zs : 1.f);
        }
        if (rem < KT) cut_steps<J>(e, rem, w.q);
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
        for (int j = J - 1; j >= 0; --j) {
            es += e[j];
            four_back([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const float ei = quad_bcast<i>(e[j]), gi = quad_bcast<i>(g[j]);
                const float* Ct = lds + (4 * j + i) * NP;
#pragma unroll
                for (int k = 0; k < NS; ++k) q[k] = fmaf(Ct[k], gi, q[k]) * __builtin_amdgcn_exp2f(ei * A2[k]);
            });
        }
        if (more) rn.put(rows[cur ^ 1]);
        __syncthreads();
    }
    es = quad_sum(es);
    if (!w.live) return;
    Part<NS> p;
#pragma unroll
    for (int k = 0; k < NS; ++k) p.v[k] = q[k];
    *part_at<NS>(a.carry, a, w, row) = p;
    if (w.q == 0) a.esum[((long long)row * a.batch + w.b) * a.d + w.ch] = es;
}

// Sums over the wave's 16 channels of v[2][4][NS] (dB | dC, step, state), through the wave's own piece of LDS: written as
// [kind, step][channel][4 NS states], read back across the channels.  Lane l adds for (kind, step) = l >> 3 the four states from
// 4 (l & 7) / SPLIT over a SPLIT-th of the channels, then SPLIT neighbouring lanes add up.  (Halving the values by lane exchanges
// instead, 24 permlane swaps and their additions for 4 steps, took 90 issue slots against 32: the vector ALUs bound this kernel.)
template <int NS> struct Sums {
    static constexpr int NP = 4 * NS, SPLIT = 8 / NS, EACH = 16 / SPLIT;
    // (16 floats more behind every EACH channels, for the SPLIT lanes that read next to each other; the whole kernel's counters show
    // 2.1 M conflict cycles for 17.3 M LDS instructions on 2048 x 8 x 2048, from which access is not known)
    static constexpr int PART = EACH * NP + 16, PITCH = SPLIT * PART;
    float lds[8 * PITCH];
    __device__ __forceinline__ void put(int block, int lane, const float* v) {
        Part<NS> p;
#pragma unroll
        for (int k = 0; k < NS; ++k) p.v[k] = v[k];
        *reinterpret_cast<Part<NS>*>(&lds[block * PITCH + (lane / (4 * EACH)) * PART + (lane % (4 * EACH)) * NS]) = p;
    }
    // -> this lane's four states' sums; block l >> 3, states from 4 * ((l & 7) / SPLIT)
    __device__ __forceinline__ f32x4 take(int lane) const {
        const float* at = &lds[(lane >> 3) * PITCH + (lane & (SPLIT - 1)) * PART + 4 * ((lane & 7) / SPLIT)];
        f32x4 s = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
        for (int c = 1; c < EACH; ++c) s += *reinterpret_cast<const f32x4*>(at + c * NP);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = s[i];
            if (SPLIT >= 2) v += quad_xor1(v);
            if (SPLIT >= 4) v += quad_xor2(v);
            if (SPLIT >= 8) {
                const float lo = dpp<0x104>(v), hi = dpp<0x114>(v);      // row_shl:4, row_shr:4: the lane with bit 2 flipped
                v += (lane & 4) ? hi : lo;
            }
            s[i] = v;
        }
        return s;
    }
};

// One tile: its states forward from the saved one, kept in registers with their factors exp(e A), then the adjoint backwards.  The
// products for dB and dC are summed over the wave's channels (Sums), over the four waves through LDS and over the channel
// tiles by scan_fold_bc_kernel, each in a fixed order; dA, dD, dbias stay in registers and leave one row per chunk and sequence.
template <typename T, int NS>
__global__ void __launch_bounds__(256, NS == 8 ? 1 : 3)
scan_bwd_kernel(ScanArgs a) {
    constexpr int KT = Tile<NS>::BACK, NP = 4 * NS, J = KT / 4;
    __shared__ __align__(16) float rows[2][2 * KT * NP];
    __shared__ __align__(16) float red[2][WAVES][2][KT][NP];
    __shared__ __align__(16) Sums<NS> sums[WAVES];
    const Where w = where(a);
    const bool b0 = w.q & 1, b1 = w.q & 2, softplus = a.softplus, gate = a.z != nullptr;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = blockIdx.z * a.chunk, last = min(a.steps, first + a.chunk), end = min(last, max(first, w.len));
    const int top = end > first ? first + ((end - first - 1) / KT) * KT : first - KT;
    float A2[NS], q[NS], dA[NS], dD = 0.f, db = 0.f;
    load_A2<NS>(a, w, A2);
    load_state<NS>(a.dstate_out, a, w, q);
    carry_in<NS>(a, w, A2, (int)gridDim.z * a.pieces - 1, ((int)blockIdx.z + 1) * a.pieces - 1, -1, q);
#pragma unroll
    for (int k = 0; k < NS; ++k) dA[k] = 0.f;
    const float Dv = a.D ? a.D[w.ch] : 0.f, bias = a.bias ? a.bias[w.ch] : 0.f;
    const long long o_t = (long long)a.batch * a.d;
    Lane<T> lx(a.x, a.x_t, a.x_b, w, top), ldt(a.dt, a.dt_t, a.dt_b, w, top), ldy(a.dy, a.dy_t, a.dy_b, w, top);
    Lane<T> lz(gate ? a.z : a.x, gate ? a.z_t : a.x_t, gate ? a.z_b : a.x_b, w, top);
    Lane<T> odx(a.dx, o_t, a.d, w, top), oddt(a.ddt, o_t, a.d, w, top), odz(a.dz, o_t, a.d, w, top);
    Rows<T, NS, KT> rn(a, w, top, true);
    const Part<NS>* ck = part_at<NS>(a.ckpt, a, w, top / KT);
    const long long ck_tile = (long long)a.batch * a.d * 4, bc_tile = (long long)KT * a.batch * a.groups * 2 * NP;
    constexpr int PER = (2 * KT * NP + 255) / 256;
    float* bc[PER];                                    // where this thread's sums of the tile go
    int bc_t[PER];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int i = threadIdx.x + 256 * r;
        bc_t[r] = i < 2 * KT * NP ? (i / NP) % KT : KT;
        bc[r] = a.part_bc + ((((long long)w.tile * a.steps + top + (i / NP) % KT) * a.batch + w.b) * a.groups + w.g) * 2 * NP + i / (KT * NP) * NP + i % NP;
    }
    {                                                  // tiles behind the sequence's end: no gradient
        const float none[J] = {};
        Lane<T> zx = odx, zdt = oddt, zz = odz;
        for (int t0 = top + KT, k = 1; t0 < last; t0 += KT, ++k) {
            const int there = left_of<KT>(a.steps, t0);
            zx.move(J);
            zdt.move(J);
            zz.move(J);
            if (w.live) {
                zx.template store_tile<J>(none, 0, there, w.q);
                zdt.template store_tile<J>(none, 0, there, w.q);
                if (gate) zz.template store_tile<J>(none, 0, there, w.q);
            }
#pragma unroll
            for (int r = 0; r < PER; ++r)
                if (bc_t[r] < there) bc[r][k * bc_tile] = 0.f;
        }
    }
    Steps<T, J> xn, dn, zn, gn;
    Part<NS> h0n;
    int rem = left_of<KT>(w.len, top);
    auto fetch = [&]() {
        rn.load(rem);
        h0n = *ck;
        xn.load(lx, rem, w.q);
        dn.load(ldt, rem, w.q);
        gn.load(ldy, rem, w.q);
        zn.load(lz, rem, w.q);
    };
    if (top >= first) {
        fetch();
        rn.put(rows[0]);
    }
    __syncthreads();
    int cur = 0;
    for (int t0 = top; t0 >= first; t0 -= KT, cur ^= 1) {
        const int now = rem, there = left_of<KT>(a.steps, t0);
        const bool more = t0 > first;
        float x[J], e[J], raw[J], g[J], dz[J], hs[KT][NS], as[KT][NS];
        const Part<NS> h0 = h0n;
        const float* lds = rows[cur] + w.q * NS;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = w.live ? to_f(xn.v[j]) : 0.f;
            raw[j] = to_f(dn.v[j]) + bias;
            const float sp = softplus_f(raw[j]), dy = w.live ? to_f(gn.v[j]) : 0.f, z = to_f(zn.v[j]), sg = sigmoid_f(z), zs = z * sg;
            e[j] = pick(softplus) ? sp : raw[j];
            g[j] = dy * (pick(gate) ? zs : 1.f);
            dz[j] = dy * (sg * (1.f + z * (1.f - sg)));
        }
        if (now < KT) cut_steps<J>(e, now, w.q);
        // the tile's states once more, and the output in front of the gate
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float u = e[j] * x[j];
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
            dz[j] *= fmaf(Dv, x[j], quad_scatter_sum(p, b0, b1));
            dD = fmaf(g[j], x[j], dD);
        }
        if (gate && w.live) odz.template store_tile<J>(dz, now, there, w.q);
        float dAt[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) dAt[k] = 0.f;
#pragma unroll
        for (int j = J - 1; j >= 0; --j) {
            float pb[4], pf[4];
            const float u = e[j] * x[j];
            four_back([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = 4 * j + i;
                const float gi = quad_bcast<i>(g[j]), ui = quad_bcast<i>(u), ei = quad_bcast<i>(e[j]);
                const float *Bt = lds + t * NP, *Ct = Bt + KT * NP;
                float vb[NS], vc[NS];
                pb[i] = pf[i] = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    q[k] = fmaf(Ct[k], gi, q[k]);
                    pb[i] = fmaf(q[k], Bt[k], pb[i]);
                    vb[k] = q[k] * ui;
                    vc[k] = gi * hs[t][k];
                    q[k] *= as[t][k];
                    const float f = q[k] * (t > 0 ? hs[t > 0 ? t - 1 : 0][k] : h0.v[k]);
                    dAt[k] = fmaf(f, ei, dAt[k]);
                    pf[i] = fmaf(f, A2[k], pf[i]);
                }
                sums[wave].put(i, lane, vb);
                sums[wave].put(4 + i, lane, vc);
            });
            wave_fence();
            const f32x4 bc_sum = sums[wave].take(lane);
            const float qb = quad_scatter_sum(pb, b0, b1), fa = quad_scatter_sum(pf, b0, b1) * LN2_F;
            const float de = fmaf(qb, x[j], fa), sl = sigmoid_f(raw[j]);
            raw[j] = de * (pick(softplus) ? sl : 1.f);                                 // now the gradient of dt
            x[j] = fmaf(g[j], Dv, qb * e[j]);                                          // now the gradient of x
            // (SPLIT lanes hold and write the same sums)
            *reinterpret_cast<f32x4*>(&red[cur][wave][lane >> 5][4 * j + ((lane >> 3) & 3)][4 * ((lane & 7) / Sums<NS>::SPLIT)]) = bc_sum;
            wave_fence();
            if (j == J / 2 && more) {                  // half of the tile's registers are free: the next one's loads
                rn.move(-1);
                ck -= ck_tile;
                lx.move(-J);
                ldt.move(-J);
                ldy.move(-J);
                lz.move(-J);
                rem = left_of<KT>(w.len, t0 - KT);
                fetch();
            }
        }
        if (now < KT) cut_steps<J>(raw, now, w.q);
#pragma unroll
        for (int j = 0; j < J; ++j) db += raw[j];
        if (w.live) {
            odx.template store_tile<J>(x, now, there, w.q);
            oddt.template store_tile<J>(raw, now, there, w.q);
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) dA[k] += dAt[k];
        if (more) rn.put(rows[cur ^ 1]);
        __syncthreads();                               // (red and rows have two sides: one barrier a tile)
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            if (bc_t[r] < there) {
                const float* at = &red[cur][0][0][0][0] + threadIdx.x + 256 * r;
                float s = at[0];
#pragma unroll
                for (int v = 1; v < WAVES; ++v) s += at[v * 2 * KT * NP];
                *bc[r] = bc_t[r] < now ? s : 0.f;      // (0 inf = NaN behind the end of a sequence whose state overflowed)
            }
            bc[r] -= bc_tile;
        }
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

// dB, dC [t][b][g][n] from the channel tiles' partial sums, in tile order; a thread takes four states
template <typename T>
__global__ void __launch_bounds__(256)
scan_fold_bc_kernel(const float* __restrict__ part, long long rows, int tiles, int np, int n, T* __restrict__ dB, T* __restrict__ dC) {
    const long long total = rows * 2 * np / 4;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int col = (int)(4 * i % (2 * np)), k = col % np;
        const f32x4* p = reinterpret_cast<const f32x4*>(part) + i;
        f32x4 s = p[0];
#pragma unroll 4
        for (int t = 1; t < tiles; ++t) s += p[t * total];
        T* to = (col < np ? dB : dC) + 4 * i / (2 * np) * n + k;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (k + c < n) to[c] = from_f<T>(s[c]);
    }
}
// dA [d][n], dD [d], dbias [d]: sums over the rows (chunks, batch elements), fp64: 16 waves take every 16th row of 64 columns, then
// wave order
__global__ void __launch_bounds__(1024)
scan_fold_params_kernel(const float* __restrict__ pa, const float* __restrict__ pd, int rows, int d, int np, int n, float* __restrict__ dA,
                        float* __restrict__ dD, float* __restrict__ db) {
    __shared__ double red[16][64];
    const int l = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long long i = (long long)blockIdx.x * 64 + l, na = (long long)d * np, all = na + 2ll * d;
    double s = 0.0;
    if (i < all) {
        const float* p = i < na ? pa + i : pd + (i - na);
        const long long row = i < na ? na : 2ll * d;
#pragma unroll 8
        for (int r = g; r < rows; r += 16) s += (double)p[r * row];
    }
    red[g][l] = s;
    __syncthreads();
    if (g != 0 || i >= all) return;
    for (int k = 1; k < 16; ++k) s += red[k][l];
    if (i < na) {
        if (i % np < n) dA[(i / np) * n + i % np] = (float)s;
    } else {
        float* to = ((i - na) & 1) ? db : dD;
        if (to) to[(i - na) >> 1] = (float)s;
    }
}

template <typename T> __device__ __forceinline__ float of_token(const void* p, long long s_b, const Where& w) {
    return p ? to_f(((const T*)p)[w.b * s_b + w.ch]) : 0.f;
}
// One token per sequence, same lanes; a lane reads its states before it writes them, so the state may be its own output.  Bound
// by launch latency: 4.3 us for 4 x 2048 x 16 (1.3 MB).
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
constexpr int SAVE_STEPS = Tile<1>::BACK;

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
    if (n > 32 || batch > 65535 || steps > (1ll << 31) - (1 << 16)) {           // (a chunk's end, rounded up to tiles, is an int too)
        jova_set_error("%s: %d states (at most 32), %lld sequences (at most 65535), %lld steps (below 2^31 - 2^16)", who, n, (long long)batch, (long long)steps);
        return JOVA_ERR_LIMIT;
    }
    return JOVA_OK;
}

ScanArgs scan_args(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* D, const void* z,
                   const float* bias, int64_t steps, int64_t batch, int d, int groups, int n, const int64_t* st, int softplus,
                   const int32_t* lengths, const float* state0) {
    ScanArgs a = {};
    a.x = x; a.dt = dt; a.A = A; a.B = B; a.C = C; a.D = D; a.z = z; a.bias = bias; a.steps = (int)steps; a.batch = (int)batch;
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
Plan fwd_plan(int64_t steps, int64_t batch, int d, int groups, int n) { return scan_plan(steps, batch, d, groups, n, FWD_TARGET, LEAST_CHUNK); }
struct BwdPlan : Plan { int pieces; long long piece; };
BwdPlan bwd_plan(int64_t steps, int64_t batch, int d, int groups, int n) {
    BwdPlan p = {scan_plan(steps, batch, d, groups, n, BWD_TARGET, LEAST_CHUNK), 1, 0};
    p.piece = p.chunk;
    if (p.chunks > 1) {
        const long long kt = tile_steps(n), wgs = (long long)channel_tiles(d, groups) * batch * (p.chunks - 1);
        long long c = FWD_TARGET / wgs;
        if (c > p.chunk / LEAST_CHUNK) c = p.chunk / LEAST_CHUNK;
        if (c > 1) p.piece = ((p.chunk + c - 1) / c + kt - 1) / kt * kt;
        p.pieces = (int)((p.chunk + p.piece - 1) / p.piece);
    }
    return p;
}

dim3 scan_grid(const ScanArgs& a, int z = 1) { return dim3((unsigned)channel_tiles(a.d, a.groups), (unsigned)a.batch, (unsigned)z); }

// Lane's 32-bit offsets: a tile of 16 steps and a channel, in bytes
bool lane_ok(const ScanArgs& a) {
    const long long lim = (1ll << 30) - a.d;
    return 16 * a.x_t < lim && 16 * a.dt_t < lim && 16 * a.z_t < lim && 16 * a.dy_t < lim && 16ll * a.batch * a.d < lim &&
           a.x_t >= 0 && a.dt_t >= 0 && a.z_t >= 0 && a.dy_t >= 0;
}
#define JOVA_SCAN_LANES(who)                                                                    \
    if (!lane_ok(a)) {                                                                          \
        jova_set_error(who ": a step of more than 2^26 elements");                          \
        return JOVA_ERR_LIMIT;                                                                  \
    }

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

#undef pick
}  // namespace

extern "C" size_t jova_selective_scan_checkpoint_bytes(int64_t steps, int64_t batch, int d, int n_state) {
    if (steps <= 0 || batch <= 0 || d < 1 || n_state < 1 || n_state > 32) return 256;
    return (size_t)((steps + SAVE_STEPS - 1) / SAVE_STEPS) * batch * d * 4 * states_per_lane(n_state) * 4;
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
    a.y = y; a.state_out = state_out_or_null; a.ckpt = (float*)checkpoints_or_null; a.chunk = (int)p.chunk;
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
BwdSpace bwd_space(int64_t steps, int64_t batch, int d, int groups, int n, const BwdPlan& p) {
    const size_t np = 4 * states_per_lane(n), rows = (size_t)p.chunks * batch * d, tiles = (d / groups + CH - 1) / CH;
    BwdSpace s;
    s.bc = 0;
    s.a = s.bc + align256(tiles * steps * batch * groups * 2 * np * 4);
    s.d = s.a + align256(rows * np * 4);
    s.carry = s.d + align256(rows * 8);
    s.esum = s.carry + align256(rows * p.pieces * np * 4);
    s.all = s.esum + align256(rows * p.pieces * 4);
    return s;
}
}  // namespace

extern "C" size_t jova_selective_scan_bwd_workspace_bytes(int64_t steps, int64_t batch, int d, int groups, int n_state) {
    if (steps < 0 || batch <= 0 || d < 1 || groups < 1 || n_state < 1 || n_state > 32) return 256;
    return bwd_space(steps, batch, d, groups, n_state, bwd_plan(steps, batch, d, groups, n_state)).all;
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
    const BwdPlan p = bwd_plan(steps, batch, d, groups, n_state);
    const BwdSpace sp = bwd_space(steps, batch, d, groups, n_state, p);
    char* ws = (char*)workspace;
    a.part_bc = (float*)(ws + sp.bc); a.part_a = (float*)(ws + sp.a); a.part_d = (float*)(ws + sp.d);
    a.carry = (float*)(ws + sp.carry); a.esum = (float*)(ws + sp.esum); a.chunk = (int)p.chunk;
    a.piece = (int)p.piece; a.pieces = p.pieces;
    a.dx = dx; a.ddt = ddt; a.dz = dz_or_null; a.dstate0 = dstate0_or_null;
    const hipStream_t s = (hipStream_t)stream;
    if (batch > 0) {
        const int rc = scan_dispatch(dtype, n_state, [&](auto t, auto k) {
            typedef decltype(t) T;
            constexpr int NS = decltype(k)::value;
            if (p.chunks > 1) {
                hipLaunchKernelGGL((scan_adjoint_kernel<T, NS>), scan_grid(a, (p.chunks - 1) * p.pieces), dim3(256), 0, s, a);
                JOVA_CHECK_LAUNCH("selective_scan_bwd (chunks)");
            }
            hipLaunchKernelGGL((scan_bwd_kernel<T, NS>), scan_grid(a, p.chunks), dim3(256), 0, s, a);
            JOVA_CHECK_LAUNCH("selective_scan_bwd");
            const long long rows = (long long)steps * batch * groups, total = rows * 2 * np / 4;
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
    hipLaunchKernelGGL(scan_fold_params_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, s, a.part_a, a.part_d,
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
