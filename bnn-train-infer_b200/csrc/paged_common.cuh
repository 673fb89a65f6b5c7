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

// The whole of one output row by one warp, straight from the definition: a
// running maximum and sum over the visible keys, the values' elements spread
// over the lanes. This is what every faster kernel has to agree with, and what
// they fall back on for a row whose masked keys hold infinities or NaN (a zero
// weight times such a value is NaN in a tensor-core product; here a masked key
// is skipped). The weights are not rounded here.
template <int D, typename T>
__device__ __noinline__ void attention_row(const AttnArgs& a, uint32_t b, const Request r, int32_t i, uint32_t head) {
    constexpr int E = D / 32;  // elements per lane
    const uint32_t lane = threadIdx.x & 31, kvh = head / a.group;
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(r.start + i) * a.q_token + (int64_t)head * a.q_head + lane * E;
    const T* kb = reinterpret_cast<const T*>(a.c.k) + (int64_t)kvh * a.c.k_head + lane * E;
    const T* vb = reinterpret_cast<const T*>(a.c.v) + (int64_t)kvh * a.c.v_head + lane * E;
    float qf[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qf[e] = to_f32<T>(q[e]);
        o[e] = 0.0f;
    }
    const int32_t pos = r.kv - r.n + i, lo = window_begin(a, pos);
    const int32_t sink_end = (int32_t)min((int64_t)a.sinks, (int64_t)lo);
    // the sum in two parts (Kahan's): one by one, 10^5 like terms would lose its last ten bits
    float m = -INFINITY, l = 0.0f, l_low = 0.0f;
    for (int32_t j = sink_end > 0 ? 0 : lo; j <= pos; ++j) {
        if (j >= sink_end && j < lo)
            j = lo;
        const int32_t page = page_of(a, b, j);
        if (page < 0) {
            j |= (1 << a.c.page_shift) - 1;  // the page's other positions too
            continue;
        }
        const int32_t row = j & ((1 << a.c.page_shift) - 1);
        const T* k = kb + (int64_t)page * a.c.k_page + (int64_t)row * a.c.k_row;
        const T* v = vb + (int64_t)page * a.c.v_page + (int64_t)row * a.c.v_row;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            s = __fmaf_rn(qf[e], to_f32<T>(k[e]), s);
#pragma unroll
        for (int d = 16; d; d >>= 1)
            s += __shfl_xor_sync(0xffffffffu, s, d);
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
        const float w = exp2_fast((m - base) * a.scale_log2);  // exactly 1 while the maximum stays
        const float p = exp2_fast((s - base) * a.scale_log2);
        const float term = __fmaf_rn(l_low, w, p), old = l * w;
        l = old + term;
        l_low = term - (l - old);
#pragma unroll
        for (int e = 0; e < E; ++e)
            o[e] = __fmaf_rn(p, to_f32<T>(v[e]), o[e] * w);
        m = mn;
    }
    const int64_t at = (int64_t)(r.start + i) * a.o_token + (int64_t)head * a.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
        store_out<T>(a, at + e, l == 0.0f ? 0.0f : o[e] / l);
    if (a.lse && lane == 0)
        a.lse[(int64_t)(r.start + i) * a.lse_token + head] = l == 0.0f ? -INFINITY : __fmaf_rn(m, a.scale, ln_fast(l));
}

}  // namespace paged
}  // namespace bnn
