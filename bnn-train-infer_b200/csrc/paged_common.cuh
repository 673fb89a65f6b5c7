// paged_common.cuh - what the paged-cache kernels share: argument blocks,
// 16-bit conversions, the geometry of a request, and the one-row attention.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bnn_device.cuh"
#include "bnn_sync.cuh"

namespace bnn {
namespace paged {

// Bits of the handle's paged status word.
constexpr int kPagedRange = 4;  // a position, slot, length, offset or max_q exceeded; kStatusTimeout: a wait expired

constexpr uint32_t kTypeF32 = 1;  // BNN_PAGED_F32

struct Cache {
    unsigned char* k;
    unsigned char* v;
    int64_t k_page, k_head, k_row;  // strides in elements
    int64_t v_page, v_head, v_row;
    uint32_t pages, kv_heads, page_shift;
};

struct AttnArgs {
    Cache c;
    const unsigned char* q;
    unsigned char* out;
    float* lse;
    const int32_t* table;
    const int32_t* kv_lens;
    const int32_t* q_starts;
    int64_t q_token, q_head, o_token, o_head, lse_token, table_stride;
    uint32_t batch, tokens, heads, group, table_width, max_q;
    uint32_t split_rows;  // most rows of a request behind a long cache that the split kernel takes
    uint32_t split_all;   // the split kernel takes every request
    uint32_t window, sinks;  // window 0: none
    uint32_t out_type;
    float scale;       // score scale
    float scale_log2;  // scale * log2(e)
    float* partials;   // workspace of the split kernel: records of partial rows
    int* group_counters;  // two for each of the split kernel's CTAs, zero between calls
    int* row_counters;    // the same
    int* status;
};

// 2^x, one MUFU operation (relative error 2^-22, subnormal results flushed:
// a weight below 2^-126 of the row's largest is zero to any 16-bit result).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) {
    return __half2float(x);
}

// Two FP32 values as one word of the 16-bit type T, each rounded to nearest.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ bool finite32(float x) { return fabsf(x) <= 3.402823466e38f; }

// One request of the call: n new tokens, the first of them token `start` of
// the batch, behind a cache of kv positions.
struct Request {
    int32_t start, n, kv;
};

// *bad: the request has tokens outside the call's, or a length that is negative
// or more than its page table holds; it is left out (n = 0) and reported.
__device__ __forceinline__ Request load_request(const AttnArgs& a, uint32_t b, bool* bad) {
    const int32_t begin = a.q_starts[b], end = a.q_starts[b + 1], kv = a.kv_lens[b];
    const int32_t room = (int32_t)min((uint64_t)a.table_width << a.c.page_shift, (uint64_t)1 << 30);
    *bad = end > begin && (begin < 0 || end > (int32_t)a.tokens || kv < 0 || kv > room);
    return Request{begin, end > begin && !*bad ? end - begin : 0, min(max(kv, 0), room)};
}

// First position of the window of a token at position p (0 without a window).
__device__ __forceinline__ int32_t window_begin(const AttnArgs& a, int32_t p) {
    return a.window ? max(p - (int32_t)a.window + 1, 0) : 0;
}

// Page of position j of request b, or -1 where the entry is no page of the pool.
__device__ __forceinline__ int32_t page_of(const AttnArgs& a, uint32_t b, int32_t j) {
    const int32_t page = a.table[(int64_t)b * a.table_stride + (j >> a.c.page_shift)];
    return (uint32_t)page < a.c.pages ? page : -1;
}

template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, float x) {
    if (a.out_type == kTypeF32)
        reinterpret_cast<float*>(a.out)[at] = x;
    else if constexpr (sizeof(T) == 2) {
        const uint32_t w = pack2<T>(x, 0.0f);
        reinterpret_cast<uint16_t*>(a.out)[at] = (uint16_t)w;
    }
}

// ln(x) for a softmax sum (one MUFU operation: off by 2^-22 at most for x near
// one, relatively elsewhere).
__device__ __forceinline__ float ln_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y * 0.693147182f;
}

// mbar_wait (bnn_sync.cuh) behind a number of plain polls: these kernels hand
// over every microsecond, and the polls that sleep and read the timer see a
// finished phase later. The slow part is out of line: there are many waits, and
// a call of few tiles runs each once.
constexpr uint32_t kQuickPolls = 64;
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kQuickPolls; ++i)
        if (mbar_try_wait(bar, parity))
            return true;
    return wait_slow(bar, parity);
}
// The same for a whole warp, which goes on as one: should the limit pass between
// two lanes' last polls, all of them give up (a part of a warp must not reach
// the next .sync instruction). The vote costs 0.5 % of an 8192-token prompt.
__device__ __noinline__ bool warp_wait_slow(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kQuickPolls; ++i)
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
            return true;
    return warp_wait_slow(bar, parity);
}

// kCount adjacent 16-bit values (2 or 4, at a multiple of their size) as FP32.
template <int kCount, typename T>
__device__ __forceinline__ void load_f32(const T* p, float* x) {
    uint32_t w[kCount / 2];
    if constexpr (kCount == 4) {
        const uint2 both = *reinterpret_cast<const uint2*>(p);
        w[0] = both.x;
        w[1] = both.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < kCount / 2; ++i) {
        const float2 f = unpack2<T>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// What the kernels fall back on for an output row that came out infinite or NaN
// behind a finite softmax sum: by one warp, straight from the definition, the
// dimensions spread over the lanes. Such a row may owe it to a value that it
// does not see (a zero weight times an infinity is NaN in a tensor-core
// product), in the positions `first` .. `last` that the kernel multiplied. Only
// the dimensions that are not finite are looked at; the others, and the sum, are
// right. Where their unseen values are all finite the row stands as it is, since
// what it sees made it so; but weights above one (kLarge) can carry a sum of
// large BF16 values past the type's end as well, and those rows are computed
// again in any case, until every wanted dimension is NaN. The weights are not
// rounded here.
//
// Eight keys at a time, so that their loads overlap: 0.19 us a key and row (0.53
// one by one), and a warp of the prompt kernel takes its rows one after another.
// A prompt of 2048 tokens, 46 us as a rule: 37 us with a NaN in a key, 0.56 ms in
// the first value (0.44 ms in F16), 12 ms in the last one or with an infinity in
// the first BF16 value. 34 ms each when every such row was computed again in full.
template <int D, typename T, bool kLarge>
__device__ __noinline__ void attention_row(const AttnArgs& a, uint32_t b, const Request r, int32_t i, uint32_t head, int32_t first,
                                           int32_t last) {
    constexpr int E = D / 32;  // elements per lane
    constexpr int kKeys = 8;
    const uint32_t lane = threadIdx.x & 31, kvh = head / a.group;
    const int32_t page_mask = (1 << a.c.page_shift) - 1;
    const int64_t at = (int64_t)(r.start + i) * a.o_token + (int64_t)head * a.o_head + lane * E;
    bool wanted[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        wanted[e] = !finite32(a.out_type == kTypeF32 ? reinterpret_cast<const float*>(a.out)[at + e]
                                                     : to_f32<T>(reinterpret_cast<const T*>(a.out)[at + e]));
    const T* kb = reinterpret_cast<const T*>(a.c.k) + (int64_t)kvh * a.c.k_head + lane * E;
    const T* vb = reinterpret_cast<const T*>(a.c.v) + (int64_t)kvh * a.c.v_head + lane * E;
    const int32_t pos = r.kv - r.n + i, lo = window_begin(a, pos);
    const int32_t sink_end = (int32_t)min((int64_t)a.sinks, (int64_t)lo);
    auto sees = [&](int32_t j) { return j <= pos && (j >= lo || j < sink_end); };

    // ---- the values that were multiplied but are not seen
    bool spoiled = false;
    for (int32_t j0 = first & -kKeys; j0 <= last && !__any_sync(0xffffffffu, spoiled); j0 += kKeys) {
        if (j0 >= lo && j0 + kKeys - 1 <= pos) {
            j0 = (pos + 1) & -kKeys;
            if (j0 > last)
                break;
        }
        const int32_t page = page_of(a, b, j0);
        if (page < 0)
            continue;
        const T* v = vb + (int64_t)page * a.c.v_page + (int64_t)(j0 & page_mask) * a.c.v_row;
        float x[kKeys][E];
#pragma unroll
        for (int u = 0; u < kKeys; ++u)
            if (j0 + u >= first && j0 + u <= last && !sees(j0 + u)) {
                load_f32<E>(v + u * a.c.v_row, x[u]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    x[u][e] = 0.0f;
            }
#pragma unroll
        for (int u = 0; u < kKeys; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e)
                spoiled |= wanted[e] && !finite32(x[u][e]);
    }
    if (!kLarge && !__any_sync(0xffffffffu, spoiled))
        return;

    // ---- the row: a running maximum and sum over the keys that it sees
    float qf[E], o[E];
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(r.start + i) * a.q_token + (int64_t)head * a.q_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qf[e] = to_f32<T>(q[e]);
        o[e] = 0.0f;
    }
    // the sum in two parts (Kahan's): one by one, 10^5 like terms would lose its last ten bits
    float m = -INFINITY, l = 0.0f, l_low = 0.0f;
    for (int32_t j0 = (sink_end > 0 ? 0 : lo) & -kKeys; j0 <= pos; j0 += kKeys) {
        if (j0 >= sink_end && j0 + kKeys - 1 < lo)
            j0 = lo & -kKeys;
        const int32_t page = page_of(a, b, j0);
        if (page < 0) {
            j0 = (j0 | page_mask) + 1 - kKeys;  // the page's other positions too
            continue;
        }
        const int64_t row = j0 & page_mask;
        const T* k = kb + (int64_t)page * a.c.k_page + row * a.c.k_row;
        const T* v = vb + (int64_t)page * a.c.v_page + row * a.c.v_row;
        float s[kKeys], x[kKeys][E];
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
            float y[E] = {};
#pragma unroll
            for (int e = 0; e < E; ++e)
                x[u][e] = 0.0f;
            if (sees(j0 + u)) {
                load_f32<E>(k + u * a.c.k_row, y);
                load_f32<E>(v + u * a.c.v_row, x[u]);
            }
            s[u] = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e)
                s[u] = __fmaf_rn(qf[e], y[e], s[u]);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1)
#pragma unroll
            for (int u = 0; u < kKeys; ++u)
                s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
        float mn = m;
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
            s[u] = sees(j0 + u) ? s[u] : -INFINITY;
            mn = fmaxf(mn, s[u]);
        }
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float w = exp2_fast((m - base) * a.scale_log2);  // exactly 1 while the maximum stays
        float term = l_low * w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            o[e] *= w;
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
            const float p = exp2_fast((s[u] - base) * a.scale_log2);
            term += p;
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[e] = __fmaf_rn(p, x[u][e], o[e]);
        }
        const float old = l * w;
        l = old + term;
        l_low = term - (l - old);
        m = mn;
        bool done = true;
#pragma unroll
        for (int e = 0; e < E; ++e)
            done = done && (!wanted[e] || isnan(o[e]));
        if (__all_sync(0xffffffffu, done))
            break;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (wanted[e])
            store_out<T>(a, at + e, l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace paged
}  // namespace bnn
