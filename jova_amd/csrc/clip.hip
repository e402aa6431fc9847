// Global norm of many gradient tensors and clipping by it (torch.nn.utils.clip_grad_norm_ semantics):
//   n = s (sum |g|^p)^(1/p) or s max |g|,   c = min(1, max_norm / (n + 1e-6)),   out = c g
// s scales the norm only (the mean over data-parallel ranks is applied by the optimizer kernel, behind the clipping).
// Two launches per JOVA_CLIP_MAX_TENSORS tensors: partial sums of every workgroup, then every workgroup of the second
// launch adds the same partial sums in the same order, so the coefficient needs no launch of its own and no atomics.
// Sums are fp64: squares of fp32 gradients up to 3e38 stay finite, and the norm does not depend on how the list is cut.
#include "seq.h"

namespace {

constexpr int MAX_T = JOVA_CLIP_MAX_TENSORS;
constexpr int BLOCKS = 1024;                           // partial sums (of all launches together: one slot each)
constexpr int CHUNK = 4096;                            // elements a workgroup takes at a time

struct TensorList {                                    // travels by value in the kernel arguments (capturable, no copy)
    const void* g[MAX_T];
    void* out[MAX_T];
    long long first[MAX_T + 1];                        // chunks before tensor i
    long long n[MAX_T];
    int count;
};

template <typename T> __device__ __forceinline__ void add_norm(float v, int kind, double& acc) {
    if (kind == 2) acc = fma((double)v, (double)v, acc);
    else if (kind == 1) acc += fabs((double)v);
    else {
        const double a = fabs((double)v);
        acc = (a > acc || a != a) ? a : acc;           // a NaN stays: nothing compares greater than it afterwards
        if (acc != acc) acc = __longlong_as_double(0x7ff8000000000000ll);
    }
}
__device__ __forceinline__ double join(double a, double b, int kind) {
    if (kind != 0) return a + b;
    return (a != a) ? a : (b > a || b != b) ? b : a;
}

__device__ __forceinline__ int find_tensor(const TensorList& l, long long chunk) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// fixed order: lanes, then waves
__device__ __forceinline__ double block_join(double v, int kind, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, 64), kind);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = join(join(red[0], red[1], kind), join(red[2], red[3], kind), kind);
    __syncthreads();
    return v;
}

template <typename T>
__global__ void __launch_bounds__(256)
grad_norm_kernel(TensorList l, int kind, double* __restrict__ part) {
    __shared__ double red[4];
    const long long chunks = l.first[l.count];
    double acc = 0.0;
    for (long long ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const int t = find_tensor(l, ch);
        const T* g = (const T*)l.g[t];
        const long long lo = (ch - l.first[t]) * CHUNK, hi = min(l.n[t], lo + CHUNK);
        for (long long i = lo + threadIdx.x; i < hi; i += 256) add_norm<T>(to_f(g[i]), kind, acc);
    }
    acc = block_join(acc, kind, red);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ float total_norm(const double* part, int n_part, int kind, float pre, double* red) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n_part; i += 256) acc = join(acc, part[i], kind);
    acc = block_join(acc, kind, red);
    return (float)((kind == 2 ? sqrt(acc) : acc) * (double)pre);
}

template <typename T>
__global__ void __launch_bounds__(256)
grad_clip_kernel(TensorList l, int kind, const double* __restrict__ part, int n_part, float pre, float max_norm,
                 float* __restrict__ norm_out, int write_all) {
    __shared__ double red[4];
    const float norm = total_norm(part, n_part, kind, pre, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float c = max_norm / (norm + 1e-6f);
    c = c < 1.f ? c : (c == c ? 1.f : c);              // (a NaN norm makes every gradient NaN, as torch does)
    if (c == 1.f && !write_all) return;                // in place and nothing to scale
    const long long chunks = l.first[l.count];
    for (long long ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const int t = find_tensor(l, ch);
        const T* g = (const T*)l.g[t];
        T* o = (T*)l.out[t];
        const long long lo = (ch - l.first[t]) * CHUNK, hi = min(l.n[t], lo + CHUNK);
        for (long long i = lo + threadIdx.x; i < hi; i += 256) o[i] = from_f<T>(to_f(g[i]) * c);
    }
}

int fill_list(TensorList& l, const void* const* g, void* const* out, const int64_t* n, int count) {
    long long at = 0;
    for (int i = 0; i < count; ++i) {
        l.g[i] = g[i];
        l.out[i] = out ? out[i] : nullptr;
        l.n[i] = n[i];
        l.first[i] = at;
        at += (n[i] + CHUNK - 1) / CHUNK;
    }
    l.first[count] = at;
    l.count = count;
    return (int)(at < BLOCKS ? (at > 0 ? at : 1) : BLOCKS);
}

int check_list(const char* who, int count, const void* const* g, const int64_t* n, int dtype, int kind) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype), "%s: unknown dtype %d", who, dtype);
    JOVA_CHECK_ARG(kind == 0 || kind == 1 || kind == 2, "%s: norm kind %d (0 = max, 1, 2)", who, kind);
    JOVA_CHECK_ARG(count >= 1 && count <= MAX_T && g && n, "%s: 1 .. %d tensors a call", who, MAX_T);
    for (int i = 0; i < count; ++i) JOVA_CHECK_ARG(n[i] >= 0 && (n[i] == 0 || g[i]), "%s: bad tensor %d", who, i);
    return JOVA_OK;
}

}  // namespace

extern "C" int jova_grad_norm_slots(void) { return BLOCKS; }

extern "C" int jova_grad_norm(int count, const void* const* grads, const int64_t* sizes, int dtype, int kind, double* slots,
                              void* stream) {
    if (const int rc = check_list("grad_norm", count, grads, sizes, dtype, kind)) return rc;
    JOVA_CHECK_ARG(slots, "grad_norm: null pointer");
    TensorList l;
    (void)fill_list(l, grads, nullptr, sizes, count);
    const hipStream_t s = (hipStream_t)stream;
    // (always BLOCKS workgroups: every slot is written, whatever the sizes)
    if (dtype == JOVA_F32) hipLaunchKernelGGL((grad_norm_kernel<float>), dim3(BLOCKS), dim3(256), 0, s, l, kind, slots);
    else if (dtype == JOVA_BF16) hipLaunchKernelGGL((grad_norm_kernel<bf16_t>), dim3(BLOCKS), dim3(256), 0, s, l, kind, slots);
    else hipLaunchKernelGGL((grad_norm_kernel<fp16_t>), dim3(BLOCKS), dim3(256), 0, s, l, kind, slots);
    JOVA_CHECK_LAUNCH("grad_norm");
    return JOVA_OK;
}

extern "C" int jova_grad_clip(int count, const void* const* grads, void* const* out, const int64_t* sizes, int dtype, int kind,
                              const double* slots, int n_slots, float norm_scale, float max_norm, float* norm_or_null, void* stream) {
    if (const int rc = check_list("grad_clip", count, grads, sizes, dtype, kind)) return rc;
    JOVA_CHECK_ARG(slots && n_slots >= 0 && out, "grad_clip: null pointer");
    for (int i = 0; i < count; ++i) JOVA_CHECK_ARG(sizes[i] == 0 || out[i], "grad_clip: bad output %d", i);
    TensorList l;
    const int blocks = fill_list(l, grads, out, sizes, count);
    int write_all = 0;
    for (int i = 0; i < count; ++i) write_all |= sizes[i] != 0 && out[i] != grads[i];
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == JOVA_F32)
        hipLaunchKernelGGL((grad_clip_kernel<float>), dim3(blocks), dim3(256), 0, s, l, kind, slots, n_slots, norm_scale, max_norm, norm_or_null, write_all);
    else if (dtype == JOVA_BF16)
        hipLaunchKernelGGL((grad_clip_kernel<bf16_t>), dim3(blocks), dim3(256), 0, s, l, kind, slots, n_slots, norm_scale, max_norm, norm_or_null, write_all);
    else
        hipLaunchKernelGGL((grad_clip_kernel<fp16_t>), dim3(blocks), dim3(256), 0, s, l, kind, slots, n_slots, norm_scale, max_norm, norm_or_null, write_all);
    JOVA_CHECK_LAUNCH("grad_clip");
    return JOVA_OK;
}
