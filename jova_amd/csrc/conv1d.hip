// Short causal depthwise convolution over time-major sequences x [T, B, D], channels independent:
//   p[t] = bias + sum_{k < W} w[k] x[t - W + 1 + k],   y[t] = p or p sigmoid(p)
// x[-1 .. -(W-1)] come from the state [W-1, B, D] (zeros without one).  A sequence may end early (lengths): what lies behind
// its end is neither read nor summed, y and the gradients there are zero, the state that is returned is the one at its end.
//   dp[t] = dy[t] or dy[t] s(p)(1 + p(1 - s(p))),  dx[t] = sum_k w[k] dp[t + W-1-k],  dw[k] = sum_{t,b} dp[t] x[t-W+1+k]
#include "seq.h"

#include <type_traits>

namespace {

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

// x[t] of channel c for t in [-(W-1), len)
template <typename T, int W>
__device__ __forceinline__ float conv_in(const ConvArgs& a, long long t, int b, int c, long long len) {
    if (t >= len) return 0.f;
    if (t >= 0) return to_f(((const T*)a.x)[t * a.x_t + b * a.x_b + c]);
    return a.state ? to_f(((const T*)a.state)[((t + W - 1) * a.batch + b) * (long long)a.d + c]) : 0.f;
}

template <typename T, int W>
__global__ void __launch_bounds__(256)
conv_fwd_kernel(ConvArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (c >= a.d) return;
    const long long len = seq_len(a, b), t0 = (long long)blockIdx.z * a.chunk, t1 = min(a.steps, t0 + a.chunk);
    float w[W], win[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = ld_any(a.weight, a.wtype, (long long)c * W + k);
    const float bias = a.bias ? ld_any(a.bias, a.wtype, c) : 0.f;
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) win[k + 1] = conv_in<T, W>(a, t0 - W + 1 + k, b, c, len);
    T* y = (T*)a.y;
    for (long long t = t0; t < t1; ++t) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) win[k] = win[k + 1];
        win[W - 1] = conv_in<T, W>(a, t, b, c, len);
        float p = bias;
#pragma unroll
        for (int k = 0; k < W; ++k) p = fmaf(w[k], win[k], p);
        if (a.silu) p *= sigmoid_f(p);
        y[(t * a.batch + b) * (long long)a.d + c] = from_f<T>(t < len ? p : 0.f);
    }
    if (a.state_out && blockIdx.z == 0) {
        T* so = (T*)a.state_out;
#pragma unroll
        for (int k = 0; k + 1 < W; ++k)
            so[((long long)k * a.batch + b) * a.d + c] = from_f<T>(conv_in<T, W>(a, len - W + 1 + k, b, c, len));
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(256)
conv_bwd_kernel(ConvArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (c >= a.d) return;
    const long long len = seq_len(a, b), t0 = (long long)blockIdx.z * a.chunk, t1 = min(a.steps, t0 + a.chunk);
    float w[W], win[W], acc[W], dw[W], db = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        w[k] = ld_any(a.weight, a.wtype, (long long)c * W + k);
        dw[k] = 0.f;
        acc[k] = 0.f;                                  // acc[j] = dx[t - W + 1 + j], complete in j = 0 after step t
    }
    const float bias = a.bias ? ld_any(a.bias, a.wtype, c) : 0.f;
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) win[k + 1] = conv_in<T, W>(a, t0 - W + 1 + k, b, c, len);
    T* dx = (T*)a.dx;
    const T *dy = (const T*)a.dy, *dso = (const T*)a.dstate_out;
    const long long lo = (a.dstate && blockIdx.z == 0) ? -(W - 1) : t0;        // chunk 0 also owns the initial state
    for (long long t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) {
            win[k] = win[k + 1];
            acc[k] = acc[k + 1];
        }
        acc[W - 1] = 0.f;
        win[W - 1] = conv_in<T, W>(a, t, b, c, len);
        if (t < len) {
            float p = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) p = fmaf(w[k], win[k], p);
            float dp = to_f(dy[t * a.dy_t + b * a.dy_b + c]);
            if (a.silu) {
                const float s = sigmoid_f(p);
                dp *= s * (1.f + p * (1.f - s));
            }
            if (t < t1) db += dp;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                acc[k] = fmaf(w[k], dp, acc[k]);
                if (t < t1) dw[k] = fmaf(dp, win[k], dw[k]);
            }
        }
        const long long s = t - W + 1;
        if (s >= lo && s < t1) {
            float v = acc[0];
            const long long j = s - (len - (W - 1));   // its place in the state that the forward returned
            if (dso && j >= 0 && s < len) v += to_f(dso[(j * a.batch + b) * a.d + c]);
            if (s >= 0) dx[(s * a.batch + b) * (long long)a.d + c] = from_f<T>(s < len ? v : 0.f);
            else ((T*)a.dstate)[((s + W - 1) * a.batch + b) * (long long)a.d + c] = from_f<T>(v);
        }
    }
    float* part = a.part + ((long long)blockIdx.z * a.batch + b) * (W + 1) * a.d + c;
#pragma unroll
    for (int k = 0; k < W; ++k) part[(long long)k * a.d] = dw[k];
    part[(long long)W * a.d] = db;
}

// dw[c][k], dbias[c] from the partial sums, rows in order
__global__ void __launch_bounds__(256)
conv_fold_kernel(const float* __restrict__ part, long long rows, int d, int width, void* __restrict__ dw, void* __restrict__ db,
                 int wtype, int accumulate) {
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = blockIdx.y, g = threadIdx.x >> 6;
    __shared__ double red[4][64];
    double s = 0.0;
    if (c < d)
        for (long long r = g; r < rows; r += 4) s += (double)part[(r * (width + 1) + k) * d + c];
    red[g][threadIdx.x & 63] = s;
    __syncthreads();
    if (g != 0 || c >= d) return;
    const int l = threadIdx.x;
    float v = (float)((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
    void* to = k < width ? dw : db;
    if (!to) return;
    const long long at = k < width ? (long long)c * width + k : c;
    if (accumulate) v += ld_any(to, wtype, at);
    st_any(to, wtype, at, v);
}

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

int conv_chunk(int64_t steps) { return 64; }

// calls f.template operator()<T, W>()
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
    if (batch > 65535 || (steps + 63) / 64 > 65535) {  // grid limits
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
    a.wtype = weight_dtype; a.chunk = conv_chunk(steps);
    const dim3 grid((d + 255) / 256, (unsigned)batch, (unsigned)(steps ? (steps + a.chunk - 1) / a.chunk : 1));
    return conv_dispatch(dtype, width, [&](auto t, auto w) {
        hipLaunchKernelGGL((conv_fwd_kernel<decltype(t), decltype(w)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
        JOVA_CHECK_LAUNCH("causal_conv_fwd");
        return JOVA_OK;
    });
}

extern "C" size_t jova_causal_conv_bwd_workspace_bytes(int64_t steps, int64_t batch, int d, int width) {
    if (steps <= 0 || batch <= 0 || d < 1 || width < 1) return 256;
    return (size_t)((steps + conv_chunk(steps) - 1) / conv_chunk(steps)) * batch * (width + 1) * d * 4;
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
    a.dx = dx; a.dstate = dstate_or_null; a.part = (float*)workspace; a.lengths = lengths_or_null;
    a.x_t = x_t; a.x_b = x_b; a.dy_t = dy_t; a.dy_b = dy_b; a.steps = steps; a.batch = (int)batch; a.d = d; a.silu = silu;
    a.wtype = weight_dtype; a.chunk = conv_chunk(steps);
    const long long chunks = (steps + a.chunk - 1) / a.chunk;
    const hipStream_t s = (hipStream_t)stream;
    if (steps > 0 && batch > 0) {
        const dim3 grid((d + 255) / 256, (unsigned)batch, (unsigned)chunks);
        const int rc = conv_dispatch(dtype, width, [&](auto t, auto w) {
            hipLaunchKernelGGL((conv_bwd_kernel<decltype(t), decltype(w)::value>), grid, dim3(256), 0, s, a);
            JOVA_CHECK_LAUNCH("causal_conv_bwd");
            return JOVA_OK;
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(conv_fold_kernel, dim3((d + 63) / 64, width + (dbias_or_null ? 1 : 0)), dim3(256), 0, s, a.part,
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
