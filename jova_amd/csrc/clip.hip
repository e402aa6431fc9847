// Global norm of many gradient tensors and clipping by it (torch.nn.utils.clip_grad_norm_ semantics):
//   n = s (sum |g|^p)^(1/p) or s max |g|,   c = min(1, max_norm / (n + 1e-6)),   out = c g
// s scales the norm only (the mean over data-parallel ranks is applied by the optimizer kernel, behind the clipping).
// Two launches for up to MAX_T tensors of a type: partial sums of every workgroup, then every workgroup of the second launch
// adds the same partial sums in the same order, so the coefficient needs no launch of its own and no atomics.
// Sums are fp64, every term by itself: squares of fp32 gradients up to 3e38 stay finite, and how the list is cut changes the norm
// by roundings of 2^-53 only.
// Bound by memory: the gradients are read twice and written once.  The second launch walks every workgroup's chunks backwards, so
// what the first one read last is still in the 256 MB cache.  400 M bf16 elements in 290 tensors: 471 us for 2.4 GB, 5.1 TB/s.
// 4 M floats in 48 tensors: 15 us on the card (5.9 + 8.9), 43 us a call: building the tensor table bounds it, on the host.
#include "seq.h"

#include <algorithm>
#include <utility>
#include <vector>

namespace {

constexpr int MAX_T = 112;                             // tensors whose table fits the 4 KB of kernel arguments
constexpr int BLOCKS = 2048;                           // workgroups of a launch at most; one partial sum each (4096: 524 us)
// A chunk is ROWS times 16 bytes a lane, 8 KB (400 M bf16 elements in 290 tensors: 4 KB 521 us, 8 KB 471, 16 KB 475; 4 M floats in
// 48: no difference).  A workgroup takes consecutive chunks, all the same number or one less.
constexpr int ROWS = 2;

struct TensorList {                                    // travels by value in the kernel arguments (capturable, no copy)
    const void* g[MAX_T];
    void* out[MAX_T];
    long long n[MAX_T];
    unsigned first[MAX_T + 1];                         // chunks before tensor i
    int count;
};

template <typename T> struct alignas(16) Vec { T v[16 / sizeof(T)]; };

template <int KIND> __device__ __forceinline__ void add_norm(float v, double& acc) {
    if (KIND == 2) acc = fma((double)v, (double)v, acc);
    else if (KIND == 1) acc += fabs((double)v);
    else {
        const double a = fabs((double)v);
        acc = (a > acc || a != a) ? a : acc;           // a NaN stays: nothing compares greater than it afterwards
    }
}
// 16 bytes at once, every term in fp64 by itself, in two chains, since an fp64 addition waits for the one before (a vector's terms
// summed in fp32 first: 400 M bf16 elements 470.4 us against 471.2)
template <int KIND, typename T> __device__ __forceinline__ void add_vec(const Vec<T>& r, double* acc) {
    constexpr int V = 16 / sizeof(T);
    if (KIND == 0) {                                   // (a maximum is the same in fp32)
        float s = 0.f;
        bool number = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = to_f(r.v[j]);
            s = fmaxf(s, fabsf(v));                    // drops a NaN
            number = number && v == v;
        }
        add_norm<0>(number ? s : __int_as_float(0x7fc00000), acc[0]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) add_norm<KIND>(to_f(r.v[j]), acc[j & 1]);
    }
}
template <int KIND> __device__ __forceinline__ double join(double a, double b) {
    if (KIND != 0) return a + b;
    return (a != a) ? a : (b > a || b != b) ? b : a;
}

__device__ __forceinline__ unsigned share(unsigned chunks, unsigned block) {
    return (unsigned)((unsigned long long)chunks * block / gridDim.x);
}
__device__ __forceinline__ int find_tensor(const TensorList& l, unsigned chunk) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// fixed order: lanes, then waves
template <int KIND> __device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<KIND>(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = join<KIND>(join<KIND>(red[0], red[1]), join<KIND>(red[2], red[3]));
    __syncthreads();
    return v;
}

// Partial sums of the workgroups' shares
template <typename T, int KIND>
__global__ void __launch_bounds__(256)
grad_norm_kernel(TensorList l, double* __restrict__ part) {
    constexpr int V = 16 / sizeof(T);
    __shared__ double red[4];
    const unsigned chunks = l.first[l.count];
    constexpr int N = ROWS * 256 * V;
    double acc[2 * ROWS] = {};
    const unsigned begin = share(chunks, blockIdx.x), end = share(chunks, blockIdx.x + 1);
    int t = find_tensor(l, begin);
    for (unsigned ch = begin; ch < end; ++ch) {
        while (l.first[t + 1] <= ch) ++t;
        const long long lo = (long long)(ch - l.first[t]) * N, n = min((long long)N, l.n[t] - lo);
        const T* g = (const T*)l.g[t] + lo;
        if (n == N && ((uintptr_t)g & 15) == 0) {
            const Vec<T>* gv = (const Vec<T>*)g + threadIdx.x;
            Vec<T> r[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) r[u] = gv[u * 256];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) add_vec<KIND, T>(r[u], acc + 2 * u);
        } else {
            const int nv = ((uintptr_t)g & 15) == 0 ? (int)n / V : 0;
            for (int i = threadIdx.x; i < nv; i += 256) add_vec<KIND, T>(((const Vec<T>*)g)[i], acc);
            for (int i = nv * V + threadIdx.x; i < n; i += 256) add_norm<KIND>(to_f(g[i]), acc[0]);
        }
    }
#pragma unroll
    for (int u = 1; u < 2 * ROWS; ++u) acc[0] = join<KIND>(acc[0], acc[u]);
    const double s = block_join<KIND>(acc[0], red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// (nontemporal stores leave the cache to the gradients that are still to be read: 481 us against 641)
template <typename T, int R> __device__ __forceinline__ void scale_rows(const Vec<T>* gv, Vec<T>* ov, float c) {
    Vec<T> r[R];
#pragma unroll
    for (int u = 0; u < R; ++u) r[u] = gv[u * 256];
#pragma unroll
    for (int u = 0; u < R; ++u) {
#pragma unroll
        for (int j = 0; j < (int)(16 / sizeof(T)); ++j) r[u].v[j] = from_f<T>(to_f(r[u].v[j]) * c);
        __builtin_nontemporal_store(*(const f32x4*)&r[u], (f32x4*)&ov[u * 256]);
    }
}

// The norm from all partial sums (every workgroup adds the same ones in the same order), then the scaling
template <typename T, int KIND>
__global__ void __launch_bounds__(256)
grad_clip_kernel(TensorList l, const double* __restrict__ part, int n_part, float pre, float max_norm, float* __restrict__ norm_out,
                 int write_all) {
    constexpr int V = 16 / sizeof(T);
    __shared__ double red[4];
    constexpr int N = ROWS * 256 * V;
    double acc = 0.0;
    for (int i = threadIdx.x; i < n_part; i += 256) acc = join<KIND>(acc, part[i]);
    acc = block_join<KIND>(acc, red);
    const float norm = (float)((KIND == 2 ? sqrt(acc) : acc) * (double)pre);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float c = max_norm / (norm + 1e-6f);
    c = c < 1.f ? c : (c == c ? 1.f : c);              // (a NaN norm makes every gradient NaN, as torch does)
    if (c == 1.f && !write_all) return;                // in place and nothing to scale
    const unsigned chunks = l.first[l.count];
    const unsigned begin = share(chunks, blockIdx.x), end = share(chunks, blockIdx.x + 1);
    if (begin == end) return;
    int t = find_tensor(l, end - 1);
    for (unsigned ch = end; ch-- > begin;) {
        while (l.first[t] > ch) --t;
        const long long lo = (long long)(ch - l.first[t]) * N, n = min((long long)N, l.n[t] - lo);
        const T* g = (const T*)l.g[t] + lo;
        T* o = (T*)l.out[t] + lo;
        if (n == N && (((uintptr_t)g | (uintptr_t)o) & 15) == 0) {
            scale_rows<T, ROWS>((const Vec<T>*)g + threadIdx.x, (Vec<T>*)o + threadIdx.x, c);
        } else {
            const int nv = (((uintptr_t)g | (uintptr_t)o) & 15) == 0 ? (int)n / V : 0;
            for (int i = threadIdx.x; i < nv; i += 256) scale_rows<T, 1>((const Vec<T>*)g + i, (Vec<T>*)o + i, c);
            for (int i = nv * V + threadIdx.x; i < n; i += 256) o[i] = from_f<T>(to_f(g[i]) * c);
        }
    }
}

struct Batch {                                         // one launch of each kernel
    int dtype, begin, end;                             // into the order of the tensors by type
};

template <typename T> int launch_norm(const TensorList& l, int blocks, int kind, double* part, hipStream_t s) {
    if (kind == 2) hipLaunchKernelGGL((grad_norm_kernel<T, 2>), dim3(blocks), dim3(256), 0, s, l, part);
    else if (kind == 1) hipLaunchKernelGGL((grad_norm_kernel<T, 1>), dim3(blocks), dim3(256), 0, s, l, part);
    else hipLaunchKernelGGL((grad_norm_kernel<T, 0>), dim3(blocks), dim3(256), 0, s, l, part);
    JOVA_CHECK_LAUNCH("clip_grads (norm)");
    return JOVA_OK;
}
template <typename T>
int launch_clip(const TensorList& l, int blocks, int kind, const double* part, int n_part, float pre, float max_norm, float* norm, int all,
                hipStream_t s) {
    if (kind == 2) hipLaunchKernelGGL((grad_clip_kernel<T, 2>), dim3(blocks), dim3(256), 0, s, l, part, n_part, pre, max_norm, norm, all);
    else if (kind == 1) hipLaunchKernelGGL((grad_clip_kernel<T, 1>), dim3(blocks), dim3(256), 0, s, l, part, n_part, pre, max_norm, norm, all);
    else hipLaunchKernelGGL((grad_clip_kernel<T, 0>), dim3(blocks), dim3(256), 0, s, l, part, n_part, pre, max_norm, norm, all);
    JOVA_CHECK_LAUNCH("clip_grads (scale)");
    return JOVA_OK;
}

int clip_all(int count, const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes, int kind,
             float norm_scale, float max_norm, float* norm, double* slots, hipStream_t s) {
    // every tensor by itself: two of the list (or an output and another's input) that share memory would race
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    std::vector<int> order;
    spans.reserve(2 * (size_t)count);
    order.reserve((size_t)count);
    for (int i = 0; i < count; ++i) {
        if (sizes[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)sizes[i] * jova_dtype_size(dtypes[i]);
        spans.emplace_back((uintptr_t)out[i], (uintptr_t)out[i] + bytes);
        if (out[i] != grads[i]) spans.emplace_back((uintptr_t)grads[i], (uintptr_t)grads[i] + bytes);
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i) JOVA_CHECK_ARG(spans[i].first >= spans[i - 1].second, "clip_grads: two tensors of the list share memory");
    std::vector<Batch> batches;
    for (int dtype = JOVA_F32; dtype <= JOVA_F16; ++dtype) {
        const int begin = (int)order.size();
        for (int i = 0; i < count; ++i)
            if (dtypes[i] == dtype && sizes[i] != 0) order.push_back(i);
        for (int b = begin; b < (int)order.size(); b += MAX_T) batches.push_back({dtype, b, std::min((int)order.size(), b + MAX_T)});
    }
    std::vector<TensorList> lists(batches.size());
    std::vector<int> blocks(batches.size());
    int n_slots = 0;
    for (size_t k = 0; k < batches.size(); ++k) {
        TensorList& l = lists[k];
        const Batch& b = batches[k];
        const long long per = ROWS * 256 * (16 / (long long)jova_dtype_size(b.dtype));
        long long at = 0;
        l.count = b.end - b.begin;
        for (int i = 0; i < l.count; ++i) {
            const int t = order[b.begin + i];
            l.g[i] = grads[t];
            l.out[i] = out[t];
            l.n[i] = sizes[t];
            l.first[i] = (unsigned)at;
            at += (sizes[t] + per - 1) / per;
        }
        if (at >= (1ll << 32) - BLOCKS) {
            jova_set_error("clip_grads: too many elements in one list");
            return JOVA_ERR_LIMIT;
        }
        l.first[l.count] = (unsigned)at;
        blocks[k] = (int)std::min<long long>(at, BLOCKS);
        double* part = slots + n_slots;
        n_slots += blocks[k];
        int rc;
        if (b.dtype == JOVA_F32) rc = launch_norm<float>(l, blocks[k], kind, part, s);
        else if (b.dtype == JOVA_BF16) rc = launch_norm<bf16_t>(l, blocks[k], kind, part, s);
        else rc = launch_norm<fp16_t>(l, blocks[k], kind, part, s);
        if (rc) return rc;
    }
    for (size_t r = batches.size(); r-- > 0;) {        // last read, first scaled
        const TensorList& l = lists[r];
        int all = 0;
        for (int i = 0; i < l.count; ++i) all |= l.out[i] != l.g[i];
        float* to = r == 0 ? norm : nullptr;
        int rc;
        if (batches[r].dtype == JOVA_F32) rc = launch_clip<float>(l, blocks[r], kind, slots, n_slots, norm_scale, max_norm, to, all, s);
        else if (batches[r].dtype == JOVA_BF16) rc = launch_clip<bf16_t>(l, blocks[r], kind, slots, n_slots, norm_scale, max_norm, to, all, s);
        else rc = launch_clip<fp16_t>(l, blocks[r], kind, slots, n_slots, norm_scale, max_norm, to, all, s);
        if (rc) return rc;
    }
    if (batches.empty()) return jova_zero_fill(norm, 4, 1, 4, s);
    return JOVA_OK;
}

}  // namespace

extern "C" size_t jova_clip_grads_workspace_bytes(int count) {
    if (count < 1) return 256;
    return (size_t)(count / MAX_T + 3) * BLOCKS * sizeof(double);              // (a type's last launch may be a short one)
}

extern "C" int jova_clip_grads(int count, const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes, int kind,
                               float norm_scale, float max_norm, float* norm, void* workspace, void* stream) {
    JOVA_CHECK_ARG(count >= 1 && grads && out && sizes && dtypes && norm && workspace, "clip_grads: bad argument");
    JOVA_CHECK_ARG(kind == 0 || kind == 1 || kind == 2, "clip_grads: norm kind %d (0 = max, 1, 2)", kind);
    for (int i = 0; i < count; ++i) {
        JOVA_CHECK_ARG(jova_dtype_ok(dtypes[i]), "clip_grads: unknown dtype %d", dtypes[i]);
        JOVA_CHECK_ARG(sizes[i] >= 0 && (sizes[i] == 0 || (grads[i] && out[i])), "clip_grads: bad tensor %d", i);
    }
    try {
        return clip_all(count, grads, out, sizes, dtypes, kind, norm_scale, max_norm, norm, (double*)workspace, (hipStream_t)stream);
    } catch (...) {                                    // host memory
        jova_set_error("clip_grads: out of host memory");
        return JOVA_ERR_LIMIT;
    }
}
