// Token embedding with scaling, and its gradient by sorted tokens.
//   y[r][:]  = s W[idx[r]][:]
//   dW[v][:] = s sum over { r : idx[r] = v } of dy[r][:], r ascending
// jova_embedding_bwd and jova_prot2vec_bwd add with float atomics, in whatever order the rows arrive; here the rows are
// first sorted by token (stable, so the rows of one token stay in ascending order), then every token's run is summed in
// that order in fp32 and rounded once: the same bits on every call.
#include "seq.h"

namespace {

constexpr int SORT_THREADS = 256;
constexpr int SORT_WAVES = SORT_THREADS / 64;
constexpr int SORT_ROUND = 2048;                       // items a workgroup ranks at a time: 8 x 64 per wave
constexpr int SORT_ITERS = SORT_ROUND / SORT_THREADS;
constexpr int SORT_MAX_BLOCKS = 1024;                  // beyond: longer spans per workgroup (the count table stays small)
constexpr int RADIX = 256;

struct SortPlan {
    int bits, passes, digit_bits, blocks;
    long long span;                                    // items per workgroup, a multiple of SORT_ROUND
};
SortPlan sort_plan(long long n, long long vocab) {
    SortPlan p;
    p.bits = 1;
    while ((1ll << p.bits) < vocab + 1) ++p.bits;      // vocab itself = "no gradient", sorts behind every token
    p.passes = (p.bits + 7) / 8;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.span = SORT_ROUND;
    while ((n + p.span - 1) / p.span > SORT_MAX_BLOCKS) p.span += SORT_ROUND;
    p.blocks = (int)((n + p.span - 1) / p.span);
    return p;
}

__device__ __forceinline__ unsigned token_key(const long long* idx, long long r, long long vocab, long long pad) {
    const long long k = idx[r];
    return (k < 0 || k >= vocab || k == pad) ? (unsigned)vocab : (unsigned)k;
}

// counts[digit][block] of this pass's digit.  Integer LDS atomics: the counts do not depend on their order.
__global__ void __launch_bounds__(SORT_THREADS)
token_hist_kernel(const long long* __restrict__ idx, const uint2* __restrict__ in, long long n, long long vocab, long long pad,
                  int shift, int mask, long long span, unsigned* __restrict__ counts) {
    __shared__ unsigned cnt[RADIX];
    for (int i = threadIdx.x; i <= mask; i += SORT_THREADS) cnt[i] = 0;
    __syncthreads();
    const long long lo = blockIdx.x * span, hi = min(n, lo + span);
    for (long long i = lo + threadIdx.x; i < hi; i += SORT_THREADS) {
        const unsigned k = idx ? token_key(idx, i, vocab, pad) : in[i].x;
        atomicAdd(&cnt[(k >> shift) & mask], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= mask; i += SORT_THREADS) counts[(long long)i * gridDim.x + blockIdx.x] = cnt[i];
}

// exclusive prefix sum of m counts in place, one workgroup
__global__ void __launch_bounds__(1024)
token_scan_kernel(unsigned* __restrict__ counts, int m) {
    __shared__ unsigned wsum[16];
    __shared__ unsigned carry;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < m; base += 1024) {
        const int i = base + threadIdx.x;
        const unsigned v = i < m ? counts[i] : 0;
        unsigned s = v;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned u = __shfl_up(s, o, 64);
            if (lane >= o) s += u;
        }
        if (lane == 63) wsum[w] = s;
        __syncthreads();
        unsigned before = carry;
        for (int k = 0; k < w; ++k) before += wsum[k];
        if (i < m) counts[i] = before + s - v;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + s;
        __syncthreads();
    }
}

// Stable scatter by this pass's digit.  Every wave owns consecutive items of the round; equal digits of 64 items find each
// other by one ballot per digit bit, so an item's rank is (earlier ones of its wave) + (peers in lower lanes), without atomics.
__global__ void __launch_bounds__(SORT_THREADS)
token_scatter_kernel(const long long* __restrict__ idx, const uint2* __restrict__ in, long long n, long long vocab, long long pad,
                     int shift, int digit_bits, long long span, const unsigned* __restrict__ counts, uint2* __restrict__ out) {
    __shared__ unsigned wcnt[SORT_WAVES][RADIX];
    __shared__ unsigned base[RADIX];
    const int radix = 1 << digit_bits, mask = radix - 1;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < radix; i += SORT_THREADS) base[i] = counts[(long long)i * gridDim.x + blockIdx.x];
    const long long lo = blockIdx.x * span, hi = min(n, lo + span);
    for (long long r0 = lo; r0 < hi; r0 += SORT_ROUND) {
        for (int i = lane; i < radix; i += 64) wcnt[w][i] = 0;
        uint2 item[SORT_ITERS];
        unsigned rank[SORT_ITERS];
#pragma unroll
        for (int it = 0; it < SORT_ITERS; ++it) {
            const long long i = r0 + w * (SORT_ROUND / SORT_WAVES) + it * 64 + lane;
            item[it] = i >= hi ? make_uint2(0, 0) : idx ? make_uint2(token_key(idx, i, vocab, pad), (unsigned)i) : in[i];
        }
        __syncthreads();                               // the round before has read wcnt and base
#pragma unroll
        for (int it = 0; it < SORT_ITERS; ++it) {
            const bool live = r0 + w * (SORT_ROUND / SORT_WAVES) + it * 64 + lane < hi;
            const unsigned dg = (item[it].x >> shift) & mask;
            unsigned long long peers = __ballot(live);
            for (int b = 0; b < digit_bits; ++b) {
                const unsigned long long bal = __ballot((dg >> b) & 1u);
                peers &= ((dg >> b) & 1u) ? bal : ~bal;
            }
            const int below = __popcll(peers & ((1ull << lane) - 1ull));
            unsigned before = 0;
            if (live) before = wcnt[w][dg];
            __builtin_amdgcn_wave_barrier();           // every lane has read its count (LDS is in order within a wave)
            if (live && below == 0) wcnt[w][dg] = before + (unsigned)__popcll(peers);
            __builtin_amdgcn_wave_barrier();
            rank[it] = before + below;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < radix; i += SORT_THREADS) {      // counts -> first places, wave by wave
            unsigned at = base[i];
            for (int k = 0; k < SORT_WAVES; ++k) {
                const unsigned c = wcnt[k][i];
                wcnt[k][i] = at;
                at += c;
            }
            base[i] = at;
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < SORT_ITERS; ++it)
            if (r0 + w * (SORT_ROUND / SORT_WAVES) + it * 64 + lane < hi)
                out[wcnt[w][(item[it].x >> shift) & mask] + rank[it]] = item[it];
        __syncthreads();
    }
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename T, int VEC>
__global__ void __launch_bounds__(256)
token_fwd_kernel(const T* __restrict__ w, const long long* __restrict__ idx, long long n, int dv, long long vocab, float scale,
                 T* __restrict__ out, int* __restrict__ bad) {
    const long long total = n * dv;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
        const long long r = e / dv;
        const int c = (int)(e - r * dv);
        const long long k = idx[r];
        Pack<T, VEC> p;
        if (k < 0 || k >= vocab) {                     // nn.Embedding raises: flag it, emit NaN
            if (c == 0) atomicOr(bad, 1);
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.v[j] = from_f<T>(__int_as_float(0x7fc00000));
        } else {
            p = reinterpret_cast<const Pack<T, VEC>*>(w)[k * dv + c];
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.v[j] = from_f<T>(to_f(p.v[j]) * scale);
        }
        reinterpret_cast<Pack<T, VEC>*>(out)[e] = p;
    }
}

// One run of equal tokens = one row of dW.  The sorted rows are cut into tiles of `tile` entries; `gw` lanes (a power of two)
// hold one tile's columns.  A run inside one tile is written at once; one that crosses a border leaves a partial sum in
// head[tile] (it began earlier) or tail[tile] (it goes on), which token_join_kernel adds up in tile order.
template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* dw, long long at, const float* acc, float scale, int accumulate) {
    Pack<T, VEC> p;
    if (accumulate) p = reinterpret_cast<const Pack<T, VEC>*>(dw)[at];
#pragma unroll
    for (int j = 0; j < VEC; ++j) p.v[j] = from_f<T>(acc[j] * scale + (accumulate ? to_f(p.v[j]) : 0.f));
    reinterpret_cast<Pack<T, VEC>*>(dw)[at] = p;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256)
token_reduce_kernel(const uint2* __restrict__ order, const T* __restrict__ dout, long long n, int dv, unsigned vocab, int tile,
                    int gw, float scale, int accumulate, T* __restrict__ dw, float* __restrict__ head, float* __restrict__ tail) {
    const int per = 256 / gw;
    const long long t = (long long)blockIdx.x * per + threadIdx.x / gw;
    const int c = blockIdx.y * 256 + threadIdx.x % gw;
    const long long e0 = t * tile;
    if (e0 >= n || c >= dv) return;
    const long long e1 = min(n, e0 + tile);
    const unsigned prev = e0 > 0 ? order[e0 - 1].x : ~0u, next = e1 < n ? order[e1].x : ~0u;
    float acc[VEC];
    unsigned cur = order[e0].x;
    bool open = cur == prev;                           // the run began in an earlier tile
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    for (long long e = e0; e <= e1; ++e) {
        const uint2 it = e < e1 ? order[e] : make_uint2(~0u, 0);
        if (it.x != cur) {
            if (cur != vocab) {
                float* part = open ? head : (e == e1 && cur == next) ? tail : nullptr;
                if (part) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) part[(t * dv + c) * VEC + j] = acc[j];
                } else {
                    write_row<T, VEC>(dw, (long long)cur * dv + c, acc, scale, accumulate);
                }
            }
            if (e == e1) return;
            cur = it.x;
            open = false;
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        }
        if (cur == vocab) return;                      // sorted behind every token: nothing follows
        const Pack<T, VEC> p = reinterpret_cast<const Pack<T, VEC>*>(dout)[(long long)it.y * dv + c];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += to_f(p.v[j]);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256)
token_join_kernel(const uint2* __restrict__ order, long long n, int dv, unsigned vocab, int tile, int gw, float scale,
                  int accumulate, T* __restrict__ dw, const float* __restrict__ head, const float* __restrict__ tail) {
    const int per = 256 / gw;
    const long long t = (long long)blockIdx.x * per + threadIdx.x / gw;
    const int c = blockIdx.y * 256 + threadIdx.x % gw;
    const long long e0 = t * tile, e1 = e0 + tile;
    if (e1 >= n || c >= dv) return;                    // the last tile has no run that goes on
    const unsigned key = order[e1 - 1].x;
    if (key == vocab || order[e1].x != key) return;
    if (order[e0].x == key && e0 > 0 && order[e0 - 1].x == key) return;      // began earlier: that tile joins it
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = tail[(t * dv + c) * VEC + j];
    for (long long u = t + 1; u * tile < n && order[u * tile].x == key; ++u) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += head[(u * dv + c) * VEC + j];
    }
    write_row<T, VEC>(dw, (long long)key * dv + c, acc, scale, accumulate);
}

__global__ void token_zero_kernel(unsigned char* __restrict__ p, long long n16, int rest) {
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n16; e += (long long)gridDim.x * blockDim.x)
        reinterpret_cast<uint4*>(p)[e] = make_uint4(0u, 0u, 0u, 0u);
    if (blockIdx.x == 0 && (int)threadIdx.x < rest) p[n16 * 16 + threadIdx.x] = 0;
}

constexpr int REDUCE_TILE = 32;
int reduce_tile(long long n) { return REDUCE_TILE; }

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int vec_of(int d, size_t esz, const void* a, const void* b) {
    int vec = (int)(16 / esz);
    while (vec > 1 && (d % vec != 0 || ((((uintptr_t)a) | ((uintptr_t)b)) & (vec * esz - 1)) != 0)) vec >>= 1;
    return vec;
}

template <typename T, int VEC>
int fwd_launch(const void* w, const int64_t* idx, int64_t n, int d, int64_t vocab, float scale, void* out, int* bad, hipStream_t s) {
    const long long total = n * (d / VEC);
    const int blocks = (int)(total + 255 < 256ll * 8192 ? (total + 255) / 256 : 8192);
    hipLaunchKernelGGL((token_fwd_kernel<T, VEC>), dim3(blocks), dim3(256), 0, s, (const T*)w, (const long long*)idx, (long long)n,
                       d / VEC, (long long)vocab, scale, (T*)out, bad);
    JOVA_CHECK_LAUNCH("token_embedding_fwd");
    return JOVA_OK;
}
template <typename T>
int fwd_dispatch(const void* w, const int64_t* idx, int64_t n, int d, int64_t vocab, float scale, void* out, int* bad, hipStream_t s) {
    switch (vec_of(d, sizeof(T), w, out)) {
        case 8: return fwd_launch<T, (sizeof(T) == 2 ? 8 : 4)>(w, idx, n, d, vocab, scale, out, bad, s);
        case 4: return fwd_launch<T, 4>(w, idx, n, d, vocab, scale, out, bad, s);
        case 2: return fwd_launch<T, 2>(w, idx, n, d, vocab, scale, out, bad, s);
        default: return fwd_launch<T, 1>(w, idx, n, d, vocab, scale, out, bad, s);
    }
}

template <typename T, int VEC>
int reduce_launch(const uint2* order, const void* dout, int64_t n, int d, int64_t vocab, float scale, int accumulate, void* dw,
                  float* head, float* tail, hipStream_t s) {
    const int dv = d / VEC, tile = reduce_tile(n);
    int gw = 8;
    while (gw < 256 && gw < dv) gw <<= 1;
    const long long tiles = (n + tile - 1) / tile;
    const dim3 grid((unsigned)((tiles + 256 / gw - 1) / (256 / gw)), (unsigned)((dv + 255) / 256));
    hipLaunchKernelGGL((token_reduce_kernel<T, VEC>), grid, dim3(256), 0, s, order, (const T*)dout, (long long)n, dv, (unsigned)vocab,
                       tile, gw, scale, accumulate, (T*)dw, head, tail);
    JOVA_CHECK_LAUNCH("token_embedding_bwd (reduce)");
    if (tiles > 1) {
        hipLaunchKernelGGL((token_join_kernel<T, VEC>), grid, dim3(256), 0, s, order, (long long)n, dv, (unsigned)vocab, tile, gw, scale,
                           accumulate, (T*)dw, head, tail);
        JOVA_CHECK_LAUNCH("token_embedding_bwd (join)");
    }
    return JOVA_OK;
}
template <typename T>
int reduce_dispatch(const uint2* order, const void* dout, int64_t n, int d, int64_t vocab, float scale, int accumulate, void* dw,
                    float* head, float* tail, hipStream_t s) {
    switch (vec_of(d, sizeof(T), dout, dw)) {
        case 8: return reduce_launch<T, (sizeof(T) == 2 ? 8 : 4)>(order, dout, n, d, vocab, scale, accumulate, dw, head, tail, s);
        case 4: return reduce_launch<T, 4>(order, dout, n, d, vocab, scale, accumulate, dw, head, tail, s);
        case 2: return reduce_launch<T, 2>(order, dout, n, d, vocab, scale, accumulate, dw, head, tail, s);
        default: return reduce_launch<T, 1>(order, dout, n, d, vocab, scale, accumulate, dw, head, tail, s);
    }
}

}  // namespace

extern "C" int jova_token_embedding_fwd(const void* weight, int dtype, const int64_t* idx, int64_t n, int d, int64_t vocab,
                                        float scale, void* out, int* bad_flag, void* stream) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype), "token_embedding_fwd: unknown dtype %d", dtype);
    JOVA_CHECK_ARG(n >= 0 && d >= 1 && vocab >= 1 && bad_flag && (n == 0 || (weight && idx && out)), "token_embedding_fwd: bad argument");
    if (n == 0) return JOVA_OK;
    if (dtype == JOVA_F32) return fwd_dispatch<float>(weight, idx, n, d, vocab, scale, out, bad_flag, (hipStream_t)stream);
    if (dtype == JOVA_BF16) return fwd_dispatch<bf16_t>(weight, idx, n, d, vocab, scale, out, bad_flag, (hipStream_t)stream);
    return fwd_dispatch<fp16_t>(weight, idx, n, d, vocab, scale, out, bad_flag, (hipStream_t)stream);
}

extern "C" size_t jova_token_embedding_bwd_workspace_bytes(int64_t n, int d, int64_t vocab) {
    if (n <= 0 || d < 1 || vocab < 1) return 256;
    const SortPlan p = sort_plan(n, vocab);
    const size_t tiles = (size_t)((n + reduce_tile(n) - 1) / reduce_tile(n));
    return 2 * align256((size_t)n * 8) + align256((size_t)RADIX * p.blocks * 4) + 2 * align256(tiles * d * 4);
}

extern "C" int jova_token_embedding_bwd(const void* dout, int dtype, const int64_t* idx, int64_t n, int d, int64_t vocab,
                                        int64_t padding_idx, float scale, void* dweight, int accumulate, void* workspace,
                                        void* stream) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype), "token_embedding_bwd: unknown dtype %d", dtype);
    JOVA_CHECK_ARG(n >= 0 && d >= 1 && vocab >= 1 && dweight && (n == 0 || (dout && idx && workspace)), "token_embedding_bwd: bad argument");
    JOVA_CHECK_ARG(n < (1ll << 31) && vocab < (1ll << 31) - 1, "token_embedding_bwd: at most 2^31 - 1 rows and tokens");
    hipStream_t s = (hipStream_t)stream;
    if (!accumulate) {
        const long long bytes = (long long)vocab * d * (long long)jova_dtype_size(dtype);
        JOVA_CHECK_ARG((((uintptr_t)dweight) & 15) == 0, "token_embedding_bwd: dweight must start on a 16-byte boundary");
        const int blocks = (int)(bytes / 16 / 256 + 1 < 8192 ? bytes / 16 / 256 + 1 : 8192);
        hipLaunchKernelGGL(token_zero_kernel, dim3(blocks), dim3(256), 0, s, (unsigned char*)dweight, bytes / 16, (int)(bytes & 15));
        JOVA_CHECK_LAUNCH("token_embedding_bwd (zero)");
    }
    if (n == 0) return JOVA_OK;
    const SortPlan p = sort_plan(n, vocab);
    char* ws = (char*)workspace;
    uint2* buf[2] = {(uint2*)ws, (uint2*)(ws + align256((size_t)n * 8))};
    ws += 2 * align256((size_t)n * 8);
    unsigned* counts = (unsigned*)ws;
    ws += align256((size_t)RADIX * p.blocks * 4);
    const int tile = reduce_tile(n);
    const size_t tiles = (size_t)((n + tile - 1) / tile);
    float* head = (float*)ws;
    float* tail = (float*)(ws + align256(tiles * d * 4));
    const int mask = (1 << p.digit_bits) - 1;
    const uint2* in = nullptr;
    for (int k = 0; k < p.passes; ++k) {
        const long long* first = k == 0 ? (const long long*)idx : nullptr;
        hipLaunchKernelGGL(token_hist_kernel, dim3(p.blocks), dim3(SORT_THREADS), 0, s, first, in, (long long)n, (long long)vocab,
                           (long long)padding_idx, k * p.digit_bits, mask, p.span, counts);
        hipLaunchKernelGGL(token_scan_kernel, dim3(1), dim3(1024), 0, s, counts, (mask + 1) * p.blocks);
        hipLaunchKernelGGL(token_scatter_kernel, dim3(p.blocks), dim3(SORT_THREADS), 0, s, first, in, (long long)n, (long long)vocab,
                           (long long)padding_idx, k * p.digit_bits, p.digit_bits, p.span, counts, buf[k & 1]);
        JOVA_CHECK_LAUNCH("token_embedding_bwd (sort)");
        in = buf[k & 1];
    }
    if (dtype == JOVA_F32) return reduce_dispatch<float>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
    if (dtype == JOVA_BF16) return reduce_dispatch<bf16_t>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
    return reduce_dispatch<fp16_t>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
}
