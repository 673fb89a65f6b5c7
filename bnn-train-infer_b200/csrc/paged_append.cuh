// paged_append.cuh - per-head RMSNorm, rotation and the append to the paged
// cache, one pass over the q|k|v rows of the new tokens.
//
// Per head of D values: y = x / sqrt(mean(x^2) + eps) * gain, then
// (a, b) -> (a cos - b sin, b cos + a sin) on the rotated pairs; FP32
// throughout, one rounding to the cache's type at the store. v is only
// converted. A head is D / 4 lanes of a warp, four adjacent values each, so
// the mean is a butterfly over those lanes, and the other value of a pair
// (i, i + rotary / 2) is rotary / 8 lanes away (adjacent pairs: in the lane).
//
// Bound: HBM for long calls (8192 tokens of 32 heads from FP32, 206 MB, 35.7 us
// = 5.8 TB/s, 88% of the measured copy rate; instruction issue 57% busy, before
// the heads of a warp were of one kind it was the limit at 53 us), the launch
// for short ones.
#pragma once

#include "paged_common.cuh"
#include "tcgen05.cuh"

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

// One warp: up to kHeads (times the heads side by side in a warp) consecutive
// heads of one kind (q, k or v) of one token; blockIdx.y counts these parts,
// the q heads' first. Two values at a time (f32x2) where both are treated alike.
template <int D, typename S, typename T, bool kInterleaved, int kHeads>
static __global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr uint32_t kLanes = D / 4;           // lanes of a head
    constexpr uint32_t kPer = 32 / kLanes;       // heads side by side in a warp
    constexpr uint32_t kPart = kHeads * kPer;
    const uint32_t lane = threadIdx.x & 31, in = lane % kLanes;
    const uint32_t t = blockIdx.x * (kAppendThreads / 32) + threadIdx.x / 32;
    griddep_launch_dependents();
    if (t >= a.tokens)
        return;
    const uint32_t q_parts = (a.heads + kPart - 1) / kPart, kv_parts = (a.c.kv_heads + kPart - 1) / kPart;
    const int which = blockIdx.y < q_parts ? 0 : blockIdx.y < q_parts + kv_parts ? 1 : 2;
    const uint32_t part = blockIdx.y - (which == 0 ? 0 : which == 1 ? q_parts : q_parts + kv_parts);
    const uint32_t heads = which == 0 ? a.heads : a.c.kv_heads;
    const uint32_t h0 = part * kPart + lane / kLanes;
    const uint32_t e0 = in * 4;  // this lane's first dimension
    griddep_wait();

    float4 x[kHeads];
    {
        const int64_t step = (int64_t)kPer * a.head[which];
        const S* p = reinterpret_cast<const S*>(a.src[which]) + (int64_t)t * a.token[which] + (int64_t)h0 * a.head[which] + e0;
        const bool aligned = ((reinterpret_cast<uintptr_t>(p) | (uint64_t)step * sizeof(S)) & (4 * sizeof(S) - 1)) == 0;
        if (aligned) {
#pragma unroll
            for (int u = 0; u < kHeads; ++u)
                x[u] = h0 + u * kPer < heads ? load4<S>(p + u * step, true) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else {
#pragma unroll
            for (int u = 0; u < kHeads; ++u)
                x[u] = h0 + u * kPer < heads ? load4<S>(p + u * step, false) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    const int32_t pos = a.positions[t], slot = a.slots[t];
    const bool pos_ok = a.rotary == 0 || (uint32_t)pos < a.table_rows;
    const int64_t room = (int64_t)a.c.pages << a.c.page_shift;
    if (blockIdx.y == 0 && lane == 0 && (!pos_ok || slot >= room))
        atomicOr(a.status, kPagedRange);

    if (which < 2) {
        // this lane's factors of the rotation
        const uint32_t half = a.rotary / 2;
        const bool turned = e0 < a.rotary && pos_ok;
        uint64_t c[2] = {f2_pack(1.0f, 1.0f), f2_pack(1.0f, 1.0f)}, s[2] = {0, 0};
        uint32_t partner = lane;
        if (turned) {
            const int64_t at = (int64_t)pos * half;
            if (kInterleaved) {
                const float2 cc = *reinterpret_cast<const float2*>(a.cos + at + e0 / 2);
                const float2 ss = *reinterpret_cast<const float2*>(a.sin + at + e0 / 2);
                c[0] = f2_pack(cc.x, cc.x);
                c[1] = f2_pack(cc.y, cc.y);
                s[0] = f2_pack(-ss.x, ss.x);
                s[1] = f2_pack(-ss.y, ss.y);
            } else {
                const bool first = e0 < half;
                const uint32_t i = first ? e0 : e0 - half;
                const float4 cc = *reinterpret_cast<const float4*>(a.cos + at + i);
                const float4 ss = *reinterpret_cast<const float4*>(a.sin + at + i);
                const float sign = first ? -1.0f : 1.0f;
                c[0] = f2_pack(cc.x, cc.y);
                c[1] = f2_pack(cc.z, cc.w);
                s[0] = f2_pack(sign * ss.x, sign * ss.y);
                s[1] = f2_pack(sign * ss.z, sign * ss.w);
                partner = first ? lane + half / 4 : lane - half / 4;
            }
        }
        // 1 / rms of each head. The heads' sums are reduced together: each exchange
        // halves the values a lane carries until one is left, so kHeads butterflies
        // cost little more than one, and one root is taken per lane
        const float* gain = a.gain[which];
        if (gain) {
            float sq[kHeads];
#pragma unroll
            for (int u = 0; u < kHeads; ++u) {
                const uint64_t lo = f2_pack(x[u].x, x[u].y), hi = f2_pack(x[u].z, x[u].w);
                const uint64_t q = f2_fma(lo, lo, f2_mul(hi, hi));
                sq[u] = f2_lo(q) + f2_hi(q);
            }
            uint32_t d = kLanes / 2;
#pragma unroll
            for (int n = kHeads; n > 1; n >>= 1, d >>= 1) {
                const bool upper = in & d;
#pragma unroll
                for (int u = 0; u < n / 2; ++u) {
                    const float keep = upper ? sq[u + n / 2] : sq[u], give = upper ? sq[u] : sq[u + n / 2];
                    sq[u] = keep + __shfl_xor_sync(0xffffffffu, give, d);
                }
            }
#pragma unroll
            for (; d; d >>= 1)
                sq[0] += __shfl_xor_sync(0xffffffffu, sq[0], d);
            const float r = rsqrtf(__fmaf_rn(sq[0], 1.0f / D, a.eps));  // off by 2 ulp: far below the 16-bit rounding
            const float4 g4 = *reinterpret_cast<const float4*>(gain + e0);
            const uint64_t g[2] = {f2_pack(g4.x, g4.y), f2_pack(g4.z, g4.w)};
#pragma unroll
            for (int u = 0; u < kHeads; ++u) {
                const float inv = __shfl_sync(0xffffffffu, r, (lane & ~(kLanes - 1u)) + u * (kLanes / kHeads));
                const uint64_t i2 = f2_pack(inv, inv);
                const uint64_t lo = f2_mul(f2_mul(f2_pack(x[u].x, x[u].y), i2), g[0]);
                const uint64_t hi = f2_mul(f2_mul(f2_pack(x[u].z, x[u].w), i2), g[1]);
                x[u] = make_float4(f2_lo(lo), f2_hi(lo), f2_lo(hi), f2_hi(hi));
            }
        }
        if (a.rotary != 0) {
#pragma unroll
            for (int u = 0; u < kHeads; ++u) {
                float4 o = make_float4(x[u].y, x[u].x, x[u].w, x[u].z);  // the pairs' other values
                if (!kInterleaved)
                    o = make_float4(__shfl_sync(0xffffffffu, x[u].x, partner), __shfl_sync(0xffffffffu, x[u].y, partner),
                                    __shfl_sync(0xffffffffu, x[u].z, partner), __shfl_sync(0xffffffffu, x[u].w, partner));
                if (turned) {
                    const uint64_t lo = f2_fma(f2_pack(x[u].x, x[u].y), c[0], f2_mul(f2_pack(o.x, o.y), s[0]));
                    const uint64_t hi = f2_fma(f2_pack(x[u].z, x[u].w), c[1], f2_mul(f2_pack(o.z, o.w), s[1]));
                    x[u] = make_float4(f2_lo(lo), f2_hi(lo), f2_lo(hi), f2_hi(hi));
                }
            }
        }
    }
    T* to;
    int64_t step;
    if (which == 0) {
        step = (int64_t)kPer * a.o_head;
        to = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.o_token + (int64_t)h0 * a.o_head + e0;
    } else {
        if (!pos_ok || slot < 0 || slot >= room)
            return;
        const int64_t page = slot >> a.c.page_shift, row = slot & ((1 << a.c.page_shift) - 1);
        const int64_t head = which == 1 ? a.c.k_head : a.c.v_head;
        step = (int64_t)kPer * head;
        to = reinterpret_cast<T*>(which == 1 ? a.c.k : a.c.v) + page * (which == 1 ? a.c.k_page : a.c.v_page) +
             row * (which == 1 ? a.c.k_row : a.c.v_row) + (int64_t)h0 * head + e0;
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u)
        if (h0 + u * kPer < heads)
            *reinterpret_cast<uint2*>(to + u * step) =
                pos_ok ? make_uint2(pack2<T>(x[u].x, x[u].y), pack2<T>(x[u].z, x[u].w)) : make_uint2(0u, 0u);
}

}  // namespace paged
}  // namespace bnn
