// Token embedding with scaling, and its gradient by sorted tokens.
//   y[r][:]  = s W[idx[r]][:]
//   dW[v][:] = s sum over { r : idx[r] = v } of dy[r][:], r ascending
// jova_embedding_bwd and jova_prot2vec_bwd add with float atomics, in whatever order the rows arrive; here the rows are
// first sorted by token (stable, so the rows of one token stay in ascending order), then every token's run is summed in fp32 and
// rounded once: ascending within tiles of 32 sorted rows, the tiles of a longer run by token_join_kernel in a fixed order that
// depends on the width and alignment of the rows.  The same bits on every call of the same shapes and alignment.
// Bound by memory (rows in, rows out, dW written whole) on long batches, by launches and the host on short ones.  65536 rows of
// 2048 bf16, 131072 tokens: 263 us for 1.34 GB = 5.1 TB/s (with cached accesses 297): lookup 84, sort with the zeros of dW 82, reduce
// 72, join 15.
// 119680 rows of 22 floats, 9049 tokens: 7 + 26 + 9 + 6 us on the card, 105 us a call (the autograd engine's thread and seven launches).
#include "seq.h"

namespace {

// Radix sort from the lowest digit.  Its time is that of its dependent launches, two a pass, not of its 8-byte items: digits as
// wide as a workgroup has threads (9 bits: 18-bit tokens in two passes; 8 bits, three passes: 326 against 304 us for the whole
// call of 65536 x 2048 bf16 and 131072 tokens), the places computed by every workgroup from all counts instead of a launch of its own.
constexpr int SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64;
// items a workgroup ranks at a time (1024 instead: 306 against 303 us)
constexpr int SORT_ITERS = 4, SORT_ROUND = SORT_THREADS * SORT_ITERS;
constexpr int SORT_MAX_BLOCKS = 128;                    // beyond: longer spans per workgroup; every one reads all counts (64: +1 .. 6 us)
constexpr int MAX_BITS = 9, RADIX = 1 << MAX_BITS;     // of a pass

struct SortPlan {
    int bits, passes, digit_bits, blocks;
    long long span;                                    // items per workgroup, a multiple of SORT_ROUND
};
SortPlan sort_plan(long long n, long long vocab) {
    SortPlan p;
    p.bits = 1;
    while ((1ll << p.bits) < vocab + 1) ++p.bits;      // vocab itself = "no gradient", sorts behind every token
    p.passes = (p.bits + MAX_BITS - 1) / MAX_BITS;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.span = ((n + SORT_MAX_BLOCKS - 1) / SORT_MAX_BLOCKS + SORT_ROUND - 1) / SORT_ROUND * SORT_ROUND;
    p.blocks = (int)((n + p.span - 1) / p.span);
    return p;
}

struct SortArgs {
    const long long* idx;                              // first pass: the tokens
    const uint2* in;                                   // later passes: (token, row)
    uint2* out;
    unsigned* counts;                                  // [block][1 << digit_bits]
    long long n, vocab, pad, span;
    int shift, digit_bits;
    // workgroups behind the sort's own fill this launch's share of dW with zeros: a sort keeps at most 128 of 256 CUs busy
    int blocks;
    uint4* zero;
    long long z0, z1;
    unsigned char* rest;                               // the last bytes of dW that are no 16
    int n_rest;
};
__device__ __forceinline__ bool zero_share(const SortArgs& a) {
    if ((int)blockIdx.x < a.blocks) return false;
    const long long step = (long long)(gridDim.x - a.blocks) * SORT_THREADS;
    for (long long i = a.z0 + (long long)((int)blockIdx.x - a.blocks) * SORT_THREADS + threadIdx.x; i < a.z1; i += step)
        a.zero[i] = make_uint4(0u, 0u, 0u, 0u);
    if ((int)blockIdx.x == a.blocks && (int)threadIdx.x < a.n_rest) a.rest[threadIdx.x] = 0;
    return true;
}
__device__ __forceinline__ uint2 sort_item(const SortArgs& a, long long i) {
    if (!a.idx) return a.in[i];
    const long long k = a.idx[i];
    return make_uint2((k < 0 || k >= a.vocab || k == a.pad) ? (unsigned)a.vocab : (unsigned)k, (unsigned)i);
}

// counts of this pass's digit.  Integer LDS atomics: the counts do not depend on their order.
__global__ void __launch_bounds__(SORT_THREADS)
token_hist_kernel(SortArgs a) {
    __shared__ unsigned cnt[RADIX];
    if (zero_share(a)) return;
    const int radix = 1 << a.digit_bits;
    if ((int)threadIdx.x < radix) cnt[threadIdx.x] = 0;
    __syncthreads();
    const long long lo = blockIdx.x * a.span, hi = min(a.n, lo + a.span);
#pragma unroll 4
    for (long long i = lo + threadIdx.x; i < hi; i += SORT_THREADS) atomicAdd(&cnt[(sort_item(a, i).x >> a.shift) & (radix - 1)], 1u);
    __syncthreads();
    if ((int)threadIdx.x < radix) a.counts[blockIdx.x * radix + threadIdx.x] = cnt[threadIdx.x];
}

// exclusive prefix sum over the workgroup's threads
__device__ __forceinline__ unsigned block_prefix(unsigned v, unsigned* wsum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(s, o, 64);
        if (lane >= o) s += u;
    }
    if (lane == 63) wsum[w] = s;
    __syncthreads();
    unsigned before = 0;
    for (int k = 0; k < w; ++k) before += wsum[k];
    __syncthreads();
    return before + s - v;
}

// Ranks one round of items: every wave owns consecutive ones; equal digits of 64 items find each other by one ballot per digit
// bit, so an item's rank is (earlier ones of its wave) + (peers in lower lanes), without atomics.  Leaves each wave's counts.
__device__ __forceinline__ void rank_round(const SortArgs& a, long long r0, long long hi, unsigned (*wcnt)[RADIX], uint2* item, unsigned* rank) {
    const int radix = 1 << a.digit_bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = lane; i < radix; i += 64) wcnt[w][i] = 0;
#pragma unroll
    for (int it = 0; it < SORT_ITERS; ++it) {
        const long long i = r0 + (w * SORT_ITERS + it) * 64 + lane;
        item[it] = i < hi ? sort_item(a, i) : make_uint2(0, 0);
    }
    wave_order();
#pragma unroll
    for (int it = 0; it < SORT_ITERS; ++it) {
        const bool live = r0 + (w * SORT_ITERS + it) * 64 + lane < hi;
        const unsigned dg = (item[it].x >> a.shift) & (radix - 1);
        unsigned long long peers = __ballot(live);
        for (int b = 0; b < a.digit_bits; ++b) {
            const unsigned long long bal = __ballot((dg >> b) & 1u);
            peers &= ((dg >> b) & 1u) ? bal : ~bal;
        }
        const int below = __popcll(peers & ((1ull << lane) - 1ull));
        unsigned before = 0;
        if (live) before = wcnt[w][dg];
        wave_order();                                  // every lane has read its count
        if (live && below == 0) wcnt[w][dg] = before + (unsigned)__popcll(peers);
        wave_order();
        rank[it] = before + below;
    }
}
__device__ __forceinline__ void place_round(const SortArgs& a, long long r0, long long hi, const unsigned (*wcnt)[RADIX], const uint2* item,
                                            const unsigned* rank) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int it = 0; it < SORT_ITERS; ++it)
        if (r0 + (w * SORT_ITERS + it) * 64 + lane < hi)
            a.out[wcnt[w][(item[it].x >> a.shift) & ((1 << a.digit_bits) - 1)] + rank[it]] = item[it];
}

// Stable scatter by this pass's digit; the places come from all workgroups' counts, read by each (at most 128 x 512)
__global__ void __launch_bounds__(SORT_THREADS)
token_scatter_kernel(SortArgs a) {
    __shared__ unsigned wcnt[SORT_WAVES][RADIX];
    __shared__ unsigned base[RADIX], total[RADIX], wsum[SORT_WAVES];
    if (zero_share(a)) return;
    const int radix = 1 << a.digit_bits, me = blockIdx.x, blocks = a.blocks;
    const int dg = threadIdx.x & (radix - 1), part = threadIdx.x >> a.digit_bits, parts = SORT_THREADS >> a.digit_bits;
    if ((int)threadIdx.x < radix) base[threadIdx.x] = total[threadIdx.x] = 0;
    __syncthreads();
    unsigned before = 0, all = 0;
#pragma unroll 8
    for (int k = part; k < blocks; k += parts) {
        const unsigned c = a.counts[k * radix + dg];
        all += c;
        before += k < me ? c : 0;
    }
    if (parts == 1) {
        base[dg] = before;
        total[dg] = all;
    } else {
        atomicAdd(&base[dg], before);                  // (integers)
        atomicAdd(&total[dg], all);
    }
    __syncthreads();
    const unsigned pre = block_prefix((int)threadIdx.x < radix ? total[threadIdx.x] : 0, wsum);
    if ((int)threadIdx.x < radix) base[threadIdx.x] += pre;
    const long long lo = me * a.span, hi = min(a.n, lo + a.span);
    uint2 item[SORT_ITERS];
    unsigned rank[SORT_ITERS];
    for (long long r0 = lo; r0 < hi; r0 += SORT_ROUND) {
        rank_round(a, r0, hi, wcnt, item, rank);
        __syncthreads();
        if ((int)threadIdx.x < radix) {                // counts -> first places, wave by wave
            unsigned at = base[threadIdx.x];
#pragma unroll
            for (int k = 0; k < SORT_WAVES; ++k) {
                const unsigned c = wcnt[k][threadIdx.x];
                wcnt[k][threadIdx.x] = at;
                at += c;
            }
            base[threadIdx.x] = at;
        }
        __syncthreads();
        place_round(a, r0, hi, wcnt, item, rank);
        __syncthreads();
    }
}

// All passes of a sort that one round holds, in one workgroup and one launch: 9 us of host time instead of 30
__global__ void __launch_bounds__(SORT_THREADS)
token_sort_small_kernel(SortArgs a, int passes, uint2* buf0, uint2* buf1) {
    __shared__ unsigned wcnt[SORT_WAVES][RADIX];
    __shared__ unsigned wsum[SORT_WAVES];
    if (zero_share(a)) return;
    const int radix = 1 << a.digit_bits;
    uint2 item[SORT_ITERS];
    unsigned rank[SORT_ITERS];
    for (int p = 0; p < passes; ++p) {
        a.shift = p * a.digit_bits;
        a.out = p & 1 ? buf1 : buf0;
        rank_round(a, 0, a.n, wcnt, item, rank);
        __syncthreads();
        unsigned all = 0;
        if ((int)threadIdx.x < radix)
#pragma unroll
            for (int k = 0; k < SORT_WAVES; ++k) all += wcnt[k][threadIdx.x];
        unsigned at = block_prefix(all, wsum);
        if ((int)threadIdx.x < radix)
#pragma unroll
            for (int k = 0; k < SORT_WAVES; ++k) {
                const unsigned c = wcnt[k][threadIdx.x];
                wcnt[k][threadIdx.x] = at;
                at += c;
            }
        __syncthreads();
        place_round(a, 0, a.n, wcnt, item, rank);
        __threadfence_block();
        __syncthreads();
        a.idx = nullptr;
        a.in = a.out;
    }
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };
template <int BYTES> struct Bits;
template <> struct Bits<2> { typedef unsigned short type; };
template <> struct Bits<4> { typedef unsigned type; };
template <> struct Bits<8> { typedef unsigned long long type; };
template <> struct Bits<16> { typedef f32x4 type; };
// what is read or written once, past the cache
template <typename P> __device__ __forceinline__ P load_once(const P* p) {
    return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const typename Bits<sizeof(P)>::type*>(p)));
}
template <typename P> __device__ __forceinline__ void store_once(P* p, const P& v) {
    typedef typename Bits<sizeof(P)>::type B;
    __builtin_nontemporal_store(__builtin_bit_cast(B, v), reinterpret_cast<B*>(p));
}

// Flat over the output's 16-byte pieces (fewer bytes where the rows or addresses do not divide), so short rows fill the lanes too.
// I: the index type that holds n * dv (64-bit divisions cost more than the row's copy).  The output goes past the cache, which then holds
// more of the table's rows: 65536 x 2048 bf16 84 us for 0.54 GB, 6.4 TB/s with the hot rows from the cache; the whole call with its gradient
// 264 us, with cached stores 276.
template <typename T, int VEC, typename I>
__global__ void __launch_bounds__(256)
token_fwd_kernel(const T* __restrict__ w, const long long* __restrict__ idx, long long n, int dv, long long vocab, float scale,
                 T* __restrict__ out, int* __restrict__ bad) {
    constexpr int U = 4;                               // rows requested before the first of them is written
    const I total = (I)(n * dv), step = (I)gridDim.x * 256;
    for (I e0 = (I)blockIdx.x * 256 + threadIdx.x; e0 < total; e0 += U * step) {
        Pack<T, VEC> p[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const I e = e0 + u * step;
            ok[u] = false;
            if (e >= total) continue;
            const I r = e / (I)dv;
            const int c = (int)(e - r * (I)dv);
            const long long k = idx[r];
            ok[u] = k >= 0 && k < vocab;
            if (ok[u]) p[u] = reinterpret_cast<const Pack<T, VEC>*>(w)[k * dv + c];
            else if (c == 0) atomicOr(bad, 1);         // nn.Embedding raises: flag it, emit NaN
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const I e = e0 + u * step;
            if (e >= total) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j) p[u].v[j] = from_f<T>(ok[u] ? to_f(p[u].v[j]) * scale : __int_as_float(0x7fc00000));
            store_once(reinterpret_cast<Pack<T, VEC>*>(out) + e, p[u]);
        }
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

// Entries of a tile: few give more rows that cross a border (16: 337 us for the whole call of 65536 x 2048 bf16, 32: 303, 64:
// 299, with 8 rows requested ahead), many leave short rows with too few workgroups (22 floats a row: 3740 tiles of 32 on 16 lanes are 234 workgroups).
constexpr int TILE = 32;
// Rows of this many 16-byte pieces (2 KB) and more are read past the cache, two ahead (more waves a SIMD); shorter ones share lines
// with each other and are latency-bound: through the cache, eight ahead.  Gradient of 65536 rows, long against short form: 1 KB
// 53 .. 56 against 53 us, 2 KB 71 against 73, 4 KB 111 against 122; 88-byte rows (119680 of them, the kernel alone) 16 against 9.
constexpr int LONG_ROW = 128;
template <typename T, int VEC, bool LONG>
__global__ void __launch_bounds__(256)
token_reduce_kernel(const uint2* __restrict__ order, const T* __restrict__ dout, long long n, int dv, unsigned vocab, int gw, float scale,
                    int accumulate, T* __restrict__ dw, float* __restrict__ head, float* __restrict__ tail) {
    constexpr int U = LONG ? 2 : 8;                    // rows requested while as many are added
    const int per = 256 / gw, g = threadIdx.x / gw;
    const long long t = (long long)blockIdx.x * per + g, e0 = t * TILE;
    const int c = blockIdx.y * 256 + threadIdx.x % gw;
    __shared__ uint2 lds[32][TILE + 2];                // a tile's entries between its neighbours' (at most 256 / 8 tiles)
    for (int i = threadIdx.x % gw; i < TILE + 2; i += gw) {
        const long long e = e0 - 1 + i;
        lds[g][i] = e >= 0 && e < n ? order[e] : make_uint2(~0u, 0);
    }
    __syncthreads();
    if (e0 >= n || c >= dv) return;
    const uint2* it = lds[g] + 1;
    const Pack<T, VEC>* rows = reinterpret_cast<const Pack<T, VEC>*>(dout) + c;
    auto row_at = [&](unsigned r) { return LONG ? load_once(rows + (long long)r * dv) : rows[(long long)r * dv]; };
    float acc[VEC];
    unsigned cur = it[0].x;
    bool open = cur == it[-1].x;                       // the run began in an earlier tile
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    Pack<T, VEC> p[U], ahead[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (it[u].x < vocab) ahead[u] = row_at(it[u].y);
    for (int e = 0; e < TILE; e += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = ahead[u];
        if (e + U < TILE)                              // in front of this batch's stores: a load behind a store waits for it
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (it[e + U + u].x < vocab) ahead[u] = row_at(it[e + U + u].y);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned key = it[e + u].x;
            if (key != cur) {                          // the run ends inside the tile
                if (cur < vocab) {
                    if (open) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) head[(t * dv + c) * VEC + j] = acc[j];
                    } else {
                        write_row<T, VEC>(dw, (long long)cur * dv + c, acc, scale, accumulate);
                    }
                }
                cur = key;
                open = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
            }
            if (key < vocab)                           // (vocab: no gradient; ~0: behind the last entry)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += to_f(p[u].v[j]);
        }
    }
    if (cur >= vocab) return;
    float* part = open ? head : it[TILE].x == cur ? tail : nullptr;
    if (part) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[(t * dv + c) * VEC + j] = acc[j];
    } else {
        write_row<T, VEC>(dw, (long long)cur * dv + c, acc, scale, accumulate);
    }
}

// The runs that cross a border: the tile a run begins in adds its tail and the heads of the tiles behind it, `parts` groups of lanes
// every parts-th tile each, then group by group.  A run's end is found by doubling and bisection over the tiles' first entries:
// most runs end in the next tile, a hot token's has thousands.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
token_join_kernel(const uint2* __restrict__ order, long long n, int dv, unsigned vocab, int gw, int parts, float scale, int accumulate,
                  T* __restrict__ dw, const float* __restrict__ head, const float* __restrict__ tail) {
    __shared__ float red[1024 * VEC];
    const int g = threadIdx.x / gw, c = blockIdx.y * 256 + threadIdx.x % gw;
    const long long t = blockIdx.x, e0 = t * TILE, e1 = e0 + TILE;       // (all conditions are the workgroup's)
    if (e1 >= n) return;                               // the last tile has no run that goes on
    const unsigned key = order[e1 - 1].x;
    if (key >= vocab || order[e1].x != key) return;
    if (e0 > 0 && order[e0 - 1].x == key) return;      // began earlier: that tile joins it
    const long long tiles = (n + TILE - 1) / TILE;
    long long last = t + 1, hi = t + 2;                // last: begins with the key; hi: does not (once found)
    for (long long by = 1; hi < tiles && order[hi * TILE].x == key; by *= 2) {
        last = hi;
        hi = last + 2 * by;
    }
    hi = min(hi, tiles);
    while (hi - last > 1) {
        const long long mid = (last + hi) >> 1;
        if (order[mid * TILE].x == key) last = mid; else hi = mid;
    }
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (c < dv) {
        if (g == 0) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = tail[(t * dv + c) * VEC + j];
        }
#pragma unroll 4
        for (long long u = t + 1 + g; u <= last; u += parts) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += head[(u * dv + c) * VEC + j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) red[j * 1024 + threadIdx.x] = acc[j];
    __syncthreads();
    if (g != 0 || c >= dv) return;
    for (int k = 1; k < parts; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += red[j * 1024 + k * gw + threadIdx.x];
    write_row<T, VEC>(dw, (long long)key * dv + c, acc, scale, accumulate);
}

__global__ void token_zero_kernel(unsigned char* __restrict__ p, long long n16, int rest) {
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n16; e += (long long)gridDim.x * blockDim.x)
        reinterpret_cast<uint4*>(p)[e] = make_uint4(0u, 0u, 0u, 0u);
    if (blockIdx.x == 0 && (int)threadIdx.x < rest) p[n16 * 16 + threadIdx.x] = 0;
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int vec_of(int d, size_t esz, const void* a, const void* b) {
    int vec = (int)(16 / esz);
    while (vec > 1 && (d % vec != 0 || ((((uintptr_t)a) | ((uintptr_t)b)) & (vec * esz - 1)) != 0)) vec >>= 1;
    return vec;
}

int gw_of(int dv) {
    int gw = 8;
    while (gw < 256 && gw < dv) gw <<= 1;
    return gw;
}

template <typename T, int VEC>
int fwd_launch(const void* w, const int64_t* idx, int64_t n, int d, int64_t vocab, float scale, void* out, int* bad, hipStream_t s) {
    const int dv = d / VEC;
    const long long total = n * dv, want = (total + 255) / 256;
    const dim3 grid((unsigned)(want < 8192 ? want : 8192));
    if (total < (1ll << 31)) hipLaunchKernelGGL((token_fwd_kernel<T, VEC, unsigned>), grid, dim3(256), 0, s, (const T*)w, (const long long*)idx,
                                                (long long)n, dv, (long long)vocab, scale, (T*)out, bad);
    else hipLaunchKernelGGL((token_fwd_kernel<T, VEC, unsigned long long>), grid, dim3(256), 0, s, (const T*)w, (const long long*)idx,
                            (long long)n, dv, (long long)vocab, scale, (T*)out, bad);
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
    const int dv = d / VEC, gw = gw_of(dv), per = 256 / gw;
    const long long tiles = (n + TILE - 1) / TILE;
    const unsigned cols = (unsigned)((dv + 255) / 256);
    const dim3 grid((unsigned)((tiles + per - 1) / per), cols);
    if (VEC * sizeof(T) == 16 && dv >= LONG_ROW)
        hipLaunchKernelGGL((token_reduce_kernel<T, VEC, VEC * sizeof(T) == 16>), grid, dim3(256), 0, s, order, (const T*)dout, (long long)n, dv,
                           (unsigned)vocab, gw, scale, accumulate, (T*)dw, head, tail);
    else
        hipLaunchKernelGGL((token_reduce_kernel<T, VEC, false>), grid, dim3(256), 0, s, order, (const T*)dout, (long long)n, dv, (unsigned)vocab,
                           gw, scale, accumulate, (T*)dw, head, tail);
    JOVA_CHECK_LAUNCH("token_embedding_bwd (reduce)");
    if (tiles > 1) {
        const int threads = gw <= 64 ? 256 : 4 * gw;
        hipLaunchKernelGGL((token_join_kernel<T, VEC>), dim3((unsigned)(tiles - 1), cols), dim3(threads), 0, s, order, (long long)n, dv,
                           (unsigned)vocab, gw, threads / gw, scale, accumulate, (T*)dw, head, tail);
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
    const size_t tiles = (size_t)((n + TILE - 1) / TILE);
    return 2 * align256((size_t)n * 8) + align256((size_t)RADIX * p.blocks * 4) + 2 * align256(tiles * d * 4);
}

extern "C" int jova_token_embedding_bwd(const void* dout, int dtype, const int64_t* idx, int64_t n, int d, int64_t vocab,
                                        int64_t padding_idx, float scale, void* dweight, int accumulate, void* workspace,
                                        void* stream) {
    JOVA_CHECK_ARG(jova_dtype_ok(dtype), "token_embedding_bwd: unknown dtype %d", dtype);
    JOVA_CHECK_ARG(n >= 0 && d >= 1 && vocab >= 1 && dweight && (n == 0 || (dout && idx && workspace)), "token_embedding_bwd: bad argument");
    JOVA_CHECK_ARG(n < (1ll << 31) && vocab < (1ll << 31) - 1, "token_embedding_bwd: at most 2^31 - 1 rows and tokens");
    const int gw_max = gw_of(d);                       // (of one element a lane; a wider one takes fewer)
    JOVA_CHECK_ARG((n + TILE - 1) / TILE * (gw_max <= 64 ? 256 : 4 * gw_max) < (1ll << 32), "token_embedding_bwd: too many rows of that width for one grid");
    hipStream_t s = (hipStream_t)stream;
    long long n16 = 0;
    int n_rest = 0;
    if (!accumulate) {
        const long long bytes = (long long)vocab * d * (long long)jova_dtype_size(dtype);
        JOVA_CHECK_ARG((((uintptr_t)dweight) & 15) == 0, "token_embedding_bwd: dweight must start on a 16-byte boundary");
        n16 = bytes / 16;
        n_rest = (int)(bytes & 15);
        if (n == 0) {
            const int blocks = (int)(n16 / 256 + 1 < 8192 ? n16 / 256 + 1 : 8192);
            hipLaunchKernelGGL(token_zero_kernel, dim3(blocks), dim3(256), 0, s, (unsigned char*)dweight, n16, n_rest);
            JOVA_CHECK_LAUNCH("token_embedding_bwd (zero)");
        }
    }
    if (n == 0) return JOVA_OK;
    const SortPlan p = sort_plan(n, vocab);
    char* ws = (char*)workspace;
    uint2* buf[2] = {(uint2*)ws, (uint2*)(ws + align256((size_t)n * 8))};
    ws += 2 * align256((size_t)n * 8);
    unsigned* counts = (unsigned*)ws;
    ws += align256((size_t)RADIX * p.blocks * 4);
    const size_t tiles = (size_t)((n + TILE - 1) / TILE);
    float* head = (float*)ws;
    float* tail = (float*)(ws + align256(tiles * d * 4));
    SortArgs a = {};
    a.idx = (const long long*)idx; a.counts = counts; a.n = n; a.vocab = vocab; a.pad = padding_idx; a.span = p.span;
    a.digit_bits = p.digit_bits; a.blocks = p.blocks; a.zero = (uint4*)dweight;
    const bool small = n <= SORT_ROUND;
    const int launches = small ? 1 : 2 * p.passes;
    int done = 0;
    // (the k-th launch's share of the zeros, and the grid that it takes: 16 x 16 bytes a lane at least)
    auto grid = [&]() {
        a.z0 = n16 * done / launches;
        a.z1 = n16 * (done + 1) / launches;
        a.n_rest = ++done == launches ? n_rest : 0;
        a.rest = (unsigned char*)dweight + n16 * 16;
        const long long zb = (a.z1 - a.z0 + 16 * SORT_THREADS - 1) / (16 * SORT_THREADS);
        return dim3((unsigned)(p.blocks + (zb < 1024 ? zb : 1024) + (zb == 0 && a.n_rest ? 1 : 0)));
    };
    const uint2* in = buf[(p.passes - 1) & 1];
    if (small) {
        const dim3 small_grid = grid();
        hipLaunchKernelGGL(token_sort_small_kernel, small_grid, dim3(SORT_THREADS), 0, s, a, p.passes, buf[0], buf[1]);
        JOVA_CHECK_LAUNCH("token_embedding_bwd (sort)");
    } else {
        for (int k = 0; k < p.passes; ++k) {
            a.shift = k * p.digit_bits;
            a.out = buf[k & 1];
            const dim3 hist_grid = grid();
            hipLaunchKernelGGL(token_hist_kernel, hist_grid, dim3(SORT_THREADS), 0, s, a);
            const dim3 scatter_grid = grid();
            hipLaunchKernelGGL(token_scatter_kernel, scatter_grid, dim3(SORT_THREADS), 0, s, a);
            JOVA_CHECK_LAUNCH("token_embedding_bwd (sort)");
            a.idx = nullptr;
            a.in = a.out;
        }
    }
    if (dtype == JOVA_F32) return reduce_dispatch<float>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
    if (dtype == JOVA_BF16) return reduce_dispatch<bf16_t>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
    return reduce_dispatch<fp16_t>(in, dout, n, d, vocab, scale, accumulate, dweight, head, tail, s);
}
