// Short causal depthwise convolution over time-major sequences x [T, B, D], channels independent:
//   p[t] = bias + sum_{k < W} w[k] x[t - W + 1 + k],   y[t] = p or p sigmoid(p)
// x[-1 .. -(W-1)] come from the state [W-1, B, D] (zeros without one).  A sequence may end early (lengths): what lies behind
// its end is neither read nor summed, y and the gradients there are zero, the state that is returned is the one at its end.
//   dp[t] = dy[t] or dy[t] s(p)(1 + p(1 - s(p))),  dx[t] = sum_k w[k] dp[t + W-1-k],  dw[k] = sum_{t,b} dp[t] x[t-W+1+k]
// Bound by memory: W multiply-adds and a sigmoid per element are far below what the vector ALUs do while it is moved; x is
// read once (the window stays in registers along the time axis), dy once, y and dx written once.
#include "seq.h"

#include <type_traits>

namespace {

// Of one thread's channels.  Few bytes and many threads hide the memory's latency better than wide accesses: forward pass of
// 8192 x 4 x 4096 bf16 with 16 bytes 142 us, 8 bytes 117, 4 bytes 108; backward pass of 232 x 128 x 512 fp32 with 8 bytes 44 us,
// 4 bytes 33 (a 4-byte thread's weights, window and sums are a quarter of the registers).
constexpr int BYTES = 4;

struct ConvArgs {
    const void *x, *dy, *weight, *bias, *state, *dstate_out;
    void *y, *dx, *state_out, *dstate;
    float* part;                                       // [rows][W + 1][D] partial sums of dw and dbias
    const int* lengths;
    long long x_t, x_b, dy_t, dy_b;
    long long steps;
    int batch, d, silu, wtype, chunk;
};

__device__ __forceinline__ long long seq_len(const ConvArgs& a, int b) {
    if (!a.lengths) return a.steps;
    const long long n = a.lengths[b];
    return n < 0 ? 0 : n > a.steps ? a.steps : n;
}

// V neighbouring channels of one step
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> none() {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = from_f<T>(0.f);
    return p;
}
// x[t] for t in [-(W-1), len), zero elsewhere
template <typename T, int W, int V>
__device__ __forceinline__ Pack<T, V> conv_in(const ConvArgs& a, long long t, int b, int c, long long len) {
    if (t >= len) return none<T, V>();
    if (t >= 0) return *(const Pack<T, V>*)((const T*)a.x + t * a.x_t + b * a.x_b + c);
    return a.state ? *(const Pack<T, V>*)((const T*)a.state + ((t + W - 1) * a.batch + b) * (long long)a.d + c) : none<T, V>();
}

// A thread owns V channels (BYTES where the rows allow it: conv_vec) of a.chunk steps and keeps the window in registers; U steps
// are loaded before the first of them is used (U = 8, 16, 32: 106.6, 104.9, 109.0 us).
// 8192 x 4 x 4096 bf16, width 4, SiLU: 104.9 us for 537 MB, 5.1 TB/s (a large copy on the same card: 5.4).
template <typename T, int W, int V>
__global__ void __launch_bounds__(256)
conv_fwd_kernel(ConvArgs a) {
    constexpr int U = 16;
    const int c = (blockIdx.x * 256 + threadIdx.x) * V, b = blockIdx.y;
    if (c >= a.d) return;
    const long long len = seq_len(a, b), t0 = (long long)blockIdx.z * a.chunk, t1 = min(a.steps, t0 + a.chunk);
    float w[V][W], bias[V], win[W][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = a.bias ? ld_any(a.bias, a.wtype, c + v) : 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) w[v][k] = ld_any(a.weight, a.wtype, (long long)(c + v) * W + k);
    }
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) {
        const Pack<T, V> p = conv_in<T, W, V>(a, t0 - W + 1 + k, b, c, len);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k + 1][v] = to_f(p.v[v]);
    }
    T* y = (T*)a.y + b * (long long)a.d + c;
    const long long y_t = (long long)a.batch * a.d;
    auto one = [&](const Pack<T, V>& in, long long t) {
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[k][v] = win[k + 1][v];
            win[W - 1][v] = to_f(in.v[v]);
            float p = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) p = fmaf(w[v][k], win[k][v], p);
            if (a.silu) p *= sigmoid_f(p);
            out.v[v] = from_f<T>(p);
        }
        *(Pack<T, V>*)(y + t * y_t) = out;
    };
    long long t = t0;
    for (; t + U <= min(t1, len); t += U) {
        const T* x = (const T*)a.x + t * a.x_t + b * a.x_b + c;
        Pack<T, V> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) in[u] = *(const Pack<T, V>*)(x + u * a.x_t);
#pragma unroll
        for (int u = 0; u < U; ++u) one(in[u], t + u);
    }
    for (; t < min(t1, len); ++t) one(conv_in<T, W, V>(a, t, b, c, len), t);
    for (; t < t1; ++t) *(Pack<T, V>*)(y + t * y_t) = none<T, V>();
    if (a.state_out && blockIdx.z == 0) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k)
            *(Pack<T, V>*)((T*)a.state_out + ((long long)k * a.batch + b) * a.d + c) = conv_in<T, W, V>(a, len - W + 1 + k, b, c, len);
    }
}

// One pass along the time axis: step t's p is computed once more from the window, dp[t] goes into the W sums of dx that it
// belongs to (acc, complete W - 1 steps later) and into the thread's dw and dbias, fp32, one row of partial sums per chunk
// and sequence (added up by conv_fold_kernel in fp64 in a fixed order: no atomics).  A chunk runs W - 1 steps past its end for dx.
// 232 x 128 x 512 fp32, ragged, width 4, SiLU: 33 us (U = 4, 8, 16: 37, 33, 38), the forward pass 19 us, the fold 4 us.
template <typename T, int W, int V>
__global__ void __launch_bounds__(256)
conv_bwd_kernel(ConvArgs a) {
    constexpr int U = 8;
    const int c = (blockIdx.x * 256 + threadIdx.x) * V, b = blockIdx.y;
    if (c >= a.d) return;
    const long long len = seq_len(a, b), t0 = (long long)blockIdx.z * a.chunk, t1 = min(a.steps, t0 + a.chunk);
    float w[V][W], bias[V], win[W][V], acc[W][V], dw[W][V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = a.bias ? ld_any(a.bias, a.wtype, c + v) : 0.f;
        db[v] = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            w[v][k] = ld_any(a.weight, a.wtype, (long long)(c + v) * W + k);
            dw[k][v] = 0.f;
            acc[k][v] = 0.f;                           // acc[j] = dx[t - W + 1 + j], complete in j = 0 after step t
        }
    }
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) {
        const Pack<T, V> p = conv_in<T, W, V>(a, t0 - W + 1 + k, b, c, len);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k + 1][v] = to_f(p.v[v]);
    }
    T* dx = (T*)a.dx + b * (long long)a.d + c;
    const long long dx_t = (long long)a.batch * a.d;
    const T *dy = (const T*)a.dy, *dso = (const T*)a.dstate_out;
    const long long lo = (a.dstate && blockIdx.z == 0) ? -(W - 1) : t0;        // chunk 0 also owns the initial state
    // step t: x[t] and dy[t] in (zeros behind the end: they add nothing), dx[t - W + 1] out; own: the step's terms of dw and dbias count
    auto one = [&](const Pack<T, V>& in, const Pack<T, V>& g, long long t, bool own, bool inner) {
        Pack<T, V> out;
        const long long s = t - W + 1, j = s - (len - (W - 1));
        Pack<T, V> so = none<T, V>();                  // gradient of the returned state, which holds x[len - W + 1 .. len)
        if (!inner && dso && j >= 0 && s < len) so = *(const Pack<T, V>*)(dso + (j * a.batch + b) * a.d + c);
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) {
                win[k][v] = win[k + 1][v];
                acc[k][v] = acc[k + 1][v];
            }
            win[W - 1][v] = to_f(in.v[v]);
            float dp = to_f(g.v[v]);
            if (a.silu) {
                float p = bias[v];
#pragma unroll
                for (int k = 0; k < W; ++k) p = fmaf(w[v][k], win[k][v], p);
                const float sg = sigmoid_f(p);
                dp *= sg * (1.f + p * (1.f - sg));
            }
            if (!inner && t >= len) dp = 0.f;
            acc[W - 1][v] = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) acc[k][v] = fmaf(w[v][k], dp, acc[k][v]);
            if (own) {
                db[v] += dp;
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k][v] = fmaf(dp, win[k][v], dw[k][v]);
            }
            out.v[v] = from_f<T>(acc[0][v] + to_f(so.v[v]));
        }
        if (s >= lo && s < t1) {
            if (s >= 0) *(Pack<T, V>*)(dx + s * dx_t) = out;
            else *(Pack<T, V>*)((T*)a.dstate + ((s + W - 1) * a.batch + b) * (long long)a.d + c) = out;
        }
    };
    long long t = t0;
    for (; t + U <= min(t1, len); t += U) {
        // the last W - 1 inputs in front of the end take the gradient of the returned state too
        const bool inner = !dso || t + U <= len - (W - 1);
        const T *x = (const T*)a.x + t * a.x_t + b * a.x_b + c, *g = dy + t * a.dy_t + b * a.dy_b + c;
        Pack<T, V> in[U], gr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            in[u] = *(const Pack<T, V>*)(x + u * a.x_t);
            gr[u] = *(const Pack<T, V>*)(g + u * a.dy_t);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(in[u], gr[u], t + u, true, inner);
    }
    for (; t < min(t1, len) + W - 1; ++t)                // (behind the end: what is left of the last W - 1 gradients)
        one(conv_in<T, W, V>(a, t, b, c, len), t < len ? *(const Pack<T, V>*)(dy + t * a.dy_t + b * a.dy_b + c) : none<T, V>(), t, t < t1, false);
    for (long long s = max(t0, len); s < t1; ++s) *(Pack<T, V>*)(dx + s * dx_t) = none<T, V>();
    if (!a.part) return;                               // (no steps: the state's gradient only)
    float* part = a.part + ((long long)blockIdx.z * a.batch + b) * (W + 1) * a.d + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < W; ++k) part[(long long)k * a.d + v] = dw[k][v];
        part[(long long)W * a.d + v] = db[v];
    }
}

// dw[c][k], dbias[c] from the partial sums: 16 waves take every 16th row of 64 channels, then wave order (4 us on 512 rows of 512
// channels: two rounds of loads and a launch)
__global__ void __launch_bounds__(1024)
conv_fold_kernel(const float* __restrict__ part, long long rows, int d, int width, void* __restrict__ dw, void* __restrict__ db,
                 int wtype, int accumulate) {
    const int l = threadIdx.x & 63, g = threadIdx.x >> 6, c = blockIdx.x * 64 + l, k = blockIdx.y;
    __shared__ double red[16][64];
    double s = 0.0;
    if (c < d) {
        const float* p = part + (long long)k * d + c;
        const long long row = (long long)(width + 1) * d;
#pragma unroll 8
        for (long long r = g; r < rows; r += 16) s += (double)p[r * row];
    }
    red[g][l] = s;
    __syncthreads();
    if (g != 0 || c >= d) return;
    for (int i = 1; i < 16; ++i) s += red[i][l];
    float v = (float)s;
    void* to = k < width ? dw : db;
    if (!to) return;
    const long long at = k < width ? (long long)c * width + k : c;
    if (accumulate) v += ld_any(to, wtype, at);
    st_any(to, wtype, at, v);
}

// One token per sequence: a thread per channel, W - 1 state rows in, moved up by one.  Every thread reads its own column before
// it writes it, so the state may be its own output.  Bound by launch latency: 3 us for 64 x 2048 (2 MB).
template <typename T, int W>
__global__ void __launch_bounds__(256)
conv_step_kernel(const T* x, long long x_b, const T* state, T* state_out, const void* weight, const void* bias, int wtype, int silu,
                 int batch, int d, T* y) {
    const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (c >= d) return;
    float win[W];
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) win[k] = to_f(state[((long long)k * batch + b) * d + c]);
    win[W - 1] = to_f(x[b * x_b + c]);
    float p = bias ? ld_any(bias, wtype, c) : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) p = fmaf(ld_any(weight, wtype, (long long)c * W + k), win[k], p);
    if (silu) p *= sigmoid_f(p);
    y[(long long)b * d + c] = from_f<T>(p);
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) state_out[((long long)k * batch + b) * d + c] = from_f<T>(win[k + 1]);
}

// Steps of a chunk: short ones give more threads, each reads (forward) or computes (backward) W - 1 steps more than it owns.
// Forward, 8192 x 4 x 4096 bf16: 16 steps 136 us, 32 104.9, 64 108, 128 114.7.  Backward with its fold, 232 x 128 x 512 fp32:
// 32 steps 37.4 us, 64 37.4, 128 48.  (Twice as long where the grid's z axis would not hold them.)
constexpr int FWD_CHUNK = 32, BWD_CHUNK = 64, MAX_GRID = 65535;

// channels a thread takes: as many as fit `bytes` and divide the rows, the strides and the addresses of all tensors, else one
int conv_vec(int dtype, int bytes, const ConvArgs& a) {
    const int es = (int)jova_dtype_size(dtype);
    int v = bytes / es;
    const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.y | (uintptr_t)a.dx | (uintptr_t)a.state | (uintptr_t)a.state_out |
                         (uintptr_t)a.dstate | (uintptr_t)a.dstate_out;
    const long long st = a.x_t | a.x_b | a.dy_t | a.dy_b | a.d;
    return (st % v == 0 && at % (uintptr_t)(v * es) == 0) ? v : 1;
}

// calls f(T(), width constant)
template <typename F> int conv_dispatch(int dtype, int width, F f) {
#define JOVA_CONV_W(W)                                                     \
    case W:                                                                \
        if (dtype == JOVA_F32) return f(float(), std::integral_constant<int, W>());   \
        if (dtype == JOVA_BF16) return f(bf16_t(), std::integral_constant<int, W>()); \
        return f(fp16_t(), std::integral_constant<int, W>());
    switch (width) {
        JOVA_CONV_W(2) JOVA_CONV_W(3) JOVA_CONV_W(4) JOVA_CONV_W(5) JOVA_CONV_W(6) JOVA_CONV_W(7) JOVA_CONV_W(8)
    }
#undef JOVA_CONV_W
    jova_set_error("causal_conv: width %d outside 2..8", width);
    return JOVA_ERR_LIMIT;
}

int conv_check(const char* who, int dtype, int wtype, int64_t steps, int64_t batch, int d, int width) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype) && jova_dtype_ok(wtype), "%s: unknown dtype", who);
    JOVA_CHECK_ARG(steps >= 0 && batch >= 0 && d >= 1, "%s: bad shape", who);
    if (width < 2 || width > 8) {
        jova_set_error("%s: width %d outside 2..8", who, width);
        return JOVA_ERR_LIMIT;
    }
    if (batch > MAX_GRID || (steps + 63) / 64 > MAX_GRID) {  // grid limits
        jova_set_error("%s: at most 65535 sequences and 65535 * 64 steps", who);
        return JOVA_ERR_LIMIT;
    }
    return JOVA_OK;
}

}  // namespace

extern "C" int jova_causal_conv_fwd(const void* x, int64_t x_t, int64_t x_b, int dtype, int64_t steps, int64_t batch, int d, int width,
                                    const void* weight, const void* bias_or_null, int weight_dtype, int silu,
                                    const int32_t* lengths_or_null, const void* state_or_null, void* y, void* state_out_or_null,
                                    void* stream) {
    if (const int rc = conv_check("causal_conv_fwd", dtype, weight_dtype, steps, batch, d, width)) return rc;
    JOVA_CHECK_ARG(weight && (steps * batch == 0 || (x && y)), "causal_conv_fwd: null pointer");
    if (batch == 0 || (steps == 0 && !state_out_or_null)) return JOVA_OK;
    ConvArgs a = {};
    a.x = x; a.weight = weight; a.bias = bias_or_null; a.state = state_or_null; a.y = y; a.state_out = state_out_or_null;
    a.lengths = lengths_or_null; a.x_t = x_t; a.x_b = x_b; a.steps = steps; a.batch = (int)batch; a.d = d; a.silu = silu;
    a.wtype = weight_dtype; a.chunk = (steps + FWD_CHUNK - 1) / FWD_CHUNK > MAX_GRID ? 2 * FWD_CHUNK : FWD_CHUNK;
    const int v = conv_vec(dtype, BYTES, a), per = 256 * v;
    const dim3 grid((d + per - 1) / per, (unsigned)batch, (unsigned)(steps ? (steps + a.chunk - 1) / a.chunk : 1));
    return conv_dispatch(dtype, width, [&](auto t, auto w) {
        typedef decltype(t) T;
        constexpr int W = decltype(w)::value;
        if (v > 1) hipLaunchKernelGGL((conv_fwd_kernel<T, W, BYTES / sizeof(T)>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((conv_fwd_kernel<T, W, 1>), grid, dim3(256), 0, (hipStream_t)stream, a);
        JOVA_CHECK_LAUNCH("causal_conv_fwd");
        return JOVA_OK;
    });
}

extern "C" size_t jova_causal_conv_bwd_workspace_bytes(int64_t steps, int64_t batch, int d, int width) {
    if (steps <= 0 || batch <= 0 || d < 1 || width < 1) return 256;
    return (size_t)((steps + BWD_CHUNK - 1) / BWD_CHUNK) * batch * (width + 1) * d * 4;
}

extern "C" int jova_causal_conv_bwd(const void* x, int64_t x_t, int64_t x_b, const void* dy, int64_t dy_t, int64_t dy_b, int dtype,
                                    int64_t steps, int64_t batch, int d, int width, const void* weight, const void* bias_or_null,
                                    int weight_dtype, int silu, const int32_t* lengths_or_null, const void* state_or_null,
                                    const void* dstate_out_or_null, void* dx, void* dweight, void* dbias_or_null, int accumulate,
                                    void* dstate_or_null, void* workspace, void* stream) {
    if (const int rc = conv_check("causal_conv_bwd", dtype, weight_dtype, steps, batch, d, width)) return rc;
    JOVA_CHECK_ARG(weight && dweight && workspace && (steps * batch == 0 || (x && dy && dx)), "causal_conv_bwd: null pointer");
    ConvArgs a = {};
    a.x = x; a.dy = dy; a.weight = weight; a.bias = bias_or_null; a.state = state_or_null; a.dstate_out = dstate_out_or_null;
    a.dx = dx; a.dstate = dstate_or_null; a.part = steps > 0 ? (float*)workspace : nullptr; a.lengths = lengths_or_null;
    a.x_t = x_t; a.x_b = x_b; a.dy_t = dy_t; a.dy_b = dy_b; a.steps = steps; a.batch = (int)batch; a.d = d; a.silu = silu;
    a.wtype = weight_dtype; a.chunk = BWD_CHUNK;
    const long long chunks = (steps + a.chunk - 1) / a.chunk;
    const hipStream_t s = (hipStream_t)stream;
    if (batch > 0 && (steps > 0 || dstate_or_null)) {  // (over no steps the state passes through, and so does its gradient)
        const int v = conv_vec(dtype, BYTES, a), per = 256 * v;
        const dim3 grid((d + per - 1) / per, (unsigned)batch, (unsigned)(chunks ? chunks : 1));
        const int rc = conv_dispatch(dtype, width, [&](auto t, auto w) {
            typedef decltype(t) T;
            constexpr int W = decltype(w)::value;
            if (v > 1) hipLaunchKernelGGL((conv_bwd_kernel<T, W, BYTES / sizeof(T)>), grid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((conv_bwd_kernel<T, W, 1>), grid, dim3(256), 0, s, a);
            JOVA_CHECK_LAUNCH("causal_conv_bwd");
            return JOVA_OK;
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(conv_fold_kernel, dim3((d + 63) / 64, width + (dbias_or_null ? 1 : 0)), dim3(1024), 0, s, (const float*)workspace,
                       (long long)(steps > 0 ? chunks * batch : 0), d, width, dweight, dbias_or_null, weight_dtype, accumulate);
    JOVA_CHECK_LAUNCH("causal_conv_bwd (fold)");
    return JOVA_OK;
}

extern "C" int jova_causal_conv_step(const void* x, int64_t x_b, const void* state, void* state_out, int dtype, int64_t batch, int d,
                                     int width, const void* weight, const void* bias_or_null, int weight_dtype, int silu, void* y,
                                     void* stream) {
    if (const int rc = conv_check("causal_conv_step", dtype, weight_dtype, 1, batch, d, width)) return rc;
    JOVA_CHECK_ARG(weight && (batch == 0 || (x && state && state_out && y)), "causal_conv_step: null pointer");
    if (batch == 0) return JOVA_OK;
    return conv_dispatch(dtype, width, [&](auto t, auto w) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((conv_step_kernel<T, decltype(w)::value>), dim3((d + 255) / 256, (unsigned)batch), dim3(256), 0,
                           (hipStream_t)stream, (const T*)x, (long long)x_b, (const T*)state, (T*)state_out, weight, bias_or_null,
                           weight_dtype, silu, (int)batch, d, (T*)y);
        JOVA_CHECK_LAUNCH("causal_conv_step");
        return JOVA_OK;
    });
}
