// paged_append.cuh - per-head RMSNorm, rotation and the append to the paged
// cache, one pass over the q|k|v rows of the new tokens.
//
// Per head of D values: y = x / sqrt(mean(x^2) + eps) * gain, then
// (a, b) -> (a cos - b sin, b cos + a sin) on the rotated pairs; FP32
// throughout, one rounding to the cache's type at the store. v is only
// converted. A head is D / 4 lanes of a warp, four adjacent values each, so
// the mean is a butterfly over those lanes, and the other value of a pair
// (i, i + rotary / 2) is rotary / 8 lanes away (adjacent pairs: in the lane).
#pragma once

#include "paged_common.cuh"

namespace bnn {
namespace paged {

struct AppendArgs {
    Cache c;
    const unsigned char* src[3];  // q, k, v
    int64_t token[3], head[3];    // strides in elements
    const float* gain[2];         // of q, k; may be nullptr
    const float* cos;
    const float* sin;
    const int32_t* positions;
    const int32_t* slots;
    unsigned char* q_out;
    int64_t o_token, o_head;
    uint32_t tokens, heads, rotary, table_rows;
    float eps;
    int* status;
};

constexpr uint32_t kAppendThreads = 128;

// Four adjacent values; `aligned`: the address is a multiple of their size.
template <typename S>
__device__ __forceinline__ float4 load4(const S* p, bool aligned) {
    if (!aligned)
        return make_float4(to_f32<S>(p[0]), to_f32<S>(p[1]), to_f32<S>(p[2]), to_f32<S>(p[3]));
    if constexpr (sizeof(S) == 4) {
        return *reinterpret_cast<const float4*>(p);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const float2 lo = unpack2<S>(w.x), hi = unpack2<S>(w.y);
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    }
}

// One warp: kHeads consecutive heads (per lane group) of one token's
// q heads, k heads, v heads in this order.
template <int D, typename S, typename T, bool kInterleaved, int kHeads>
static __global__ void __launch_bounds__(kAppendThreads) append_kernel(AppendArgs a) {
    constexpr int kLanes = D / 4;           // lanes of a head
    constexpr int kPer = 32 / kLanes;       // heads side by side in a warp
    const uint32_t lane = threadIdx.x & 31, in = lane % kLanes;
    const uint32_t all = a.heads + 2 * a.c.kv_heads;
    const uint32_t parts = (all + kHeads * kPer - 1) / (kHeads * kPer);
    const uint32_t warp = blockIdx.x * (kAppendThreads / 32) + threadIdx.x / 32;
    const uint32_t t = warp / parts;
    griddep_launch_dependents();
    if (t >= a.tokens)
        return;
    const uint32_t h0 = (warp % parts) * (kHeads * kPer) + lane / kLanes;
    griddep_wait();
    const int32_t pos = a.positions[t], slot = a.slots[t];
    const bool pos_ok = a.rotary == 0 || (uint32_t)pos < a.table_rows;
    const int64_t room = (int64_t)a.c.pages << a.c.page_shift;
    const bool stored = pos_ok && slot >= 0 && slot < room;
    if (lane == 0 && (!pos_ok || slot >= room))
        atomicOr(a.status, kPagedRange);
    const uint32_t e0 = in * 4;  // this lane's first dimension

    float4 x[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
        const uint32_t h = h0 + u * kPer;
        if (h < all) {
            const int which = h < a.heads ? 0 : h < a.heads + a.c.kv_heads ? 1 : 2;
            const uint32_t hh = which == 0 ? h : which == 1 ? h - a.heads : h - a.heads - a.c.kv_heads;
            const S* p = reinterpret_cast<const S*>(a.src[which]) + (int64_t)t * a.token[which] +
                         (int64_t)hh * a.head[which] + e0;
            x[u] = load4<S>(p, (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(S) - 1)) == 0);
        } else {
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    // this lane's factors of the rotation
    const uint32_t half = a.rotary / 2;
    const bool turned = e0 < a.rotary && pos_ok;
    float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t partner = lane;
    if (turned) {
        const int64_t at = (int64_t)pos * half;
        if (kInterleaved) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                c[2 * e] = c[2 * e + 1] = a.cos[at + e0 / 2 + e];
                s[2 * e + 1] = a.sin[at + e0 / 2 + e];
                s[2 * e] = -s[2 * e + 1];
            }
        } else {
            const bool first = e0 < half;
            const uint32_t i = first ? e0 : e0 - half;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = a.cos[at + i + e];
                s[e] = first ? -a.sin[at + i + e] : a.sin[at + i + e];
            }
            partner = first ? lane + half / 4 : lane - half / 4;
        }
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
        const uint32_t h = h0 + u * kPer;
        const int which = h < a.heads ? 0 : h < a.heads + a.c.kv_heads ? 1 : 2;
        float4 y = x[u];
        const float* gain = which < 2 ? a.gain[which] : nullptr;
        float sq = __fmaf_rn(y.x, y.x, __fmaf_rn(y.y, y.y, __fmaf_rn(y.z, y.z, y.w * y.w)));
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1)
            sq += __shfl_xor_sync(0xffffffffu, sq, d);
        if (gain) {
            const float4 g = *reinterpret_cast<const float4*>(gain + e0);
            const float inv = 1.0f / sqrtf(__fmaf_rn(sq, 1.0f / D, a.eps));
            y = make_float4(y.x * inv * g.x, y.y * inv * g.y, y.z * inv * g.z, y.w * inv * g.w);
        }
        float4 o = make_float4(y.y, y.x, y.w, y.z);  // the pairs' other values
        if (!kInterleaved) {
            o.x = __shfl_sync(0xffffffffu, y.x, partner);
            o.y = __shfl_sync(0xffffffffu, y.y, partner);
            o.z = __shfl_sync(0xffffffffu, y.z, partner);
            o.w = __shfl_sync(0xffffffffu, y.w, partner);
        }
        if (which < 2 && turned)
            y = make_float4(__fmaf_rn(y.x, c[0], o.x * s[0]), __fmaf_rn(y.y, c[1], o.y * s[1]),
                            __fmaf_rn(y.z, c[2], o.z * s[2]), __fmaf_rn(y.w, c[3], o.w * s[3]));
        if (h >= all)
            continue;
        uint2 w = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
        if (which == 0) {
            if (!pos_ok)
                w = make_uint2(0u, 0u);
            T* p = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.o_token + (int64_t)h * a.o_head + e0;
            *reinterpret_cast<uint2*>(p) = w;
        } else if (stored) {
            const uint32_t hh = which == 1 ? h - a.heads : h - a.heads - a.c.kv_heads;
            const int64_t page = slot >> a.c.page_shift, row = slot & ((1 << a.c.page_shift) - 1);
            const int64_t at = which == 1 ? page * a.c.k_page + (int64_t)hh * a.c.k_head + row * a.c.k_row
                                          : page * a.c.v_page + (int64_t)hh * a.c.v_head + row * a.c.v_row;
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(which == 1 ? a.c.k : a.c.v) + at + e0) = w;
        }
    }
}

}  // namespace paged
}  // namespace bnn
