// paged_decode.cuh - attention of a few new tokens per request over its pages,
// split over the cache's length and joined.
//
// For one KV head of one request (a "row" below) the group's query heads and
// new tokens are the 16 rows of an m16n8k16 product: S = Q K^T for 16 keys,
// P = 2^(c (S - m)) with the running maximum m, O = O 2^(c (m_old - m)) + P V,
// l likewise; partial (m, l, O) of disjoint key ranges join as
// O = sum_p 2^(c (m_p - M)) O_p / sum_p 2^(c (m_p - M)) l_p.
//
// Bound: HBM, each visible K and V row is read once. The whole call's keys are
// one sequence of 64-key blocks (request by request, head by head), cut into
// equal shares, one per CTA, so requests of unlike lengths load every SM alike;
// a row that falls into several shares is joined by the CTA that finishes it
// last, in the order of the shares (the result does not depend on timing), and
// rows of at most kWholeBlocks blocks are not cut. Each warp streams its own
// 16-key tiles through a ring of cp.async stages: no CTA barrier inside a row.
#pragma once

#include <type_traits>

#include "paged_common.cuh"

namespace bnn {
namespace paged {

constexpr uint32_t kDecWarps = 4;
constexpr uint32_t kDecThreads = kDecWarps * 32;
constexpr uint32_t kDecTile = 16;                        // keys of a warp's step
constexpr uint32_t kDecBlock = kDecTile * kDecWarps;     // keys of a CTA's step
constexpr uint32_t kDecPerSm = 2;                        // CTAs an SM holds
constexpr uint32_t kWholeBlocks = 8;
constexpr uint32_t kMinShare = 4;                        // blocks
constexpr uint32_t kDecRows = 16;

template <int D>
struct DecodeShape {
    static constexpr uint32_t kStageBytes = 2 * kDecTile * D * 2;  // K and V rows of a tile
    static constexpr uint32_t kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kWarpBytes = kStages * kStageBytes;
    static constexpr uint32_t kRingBytes = kDecWarps * kWarpBytes;
    static constexpr uint32_t kRecord = kDecRows * (D + 2);  // floats of a partial: m[16], l[16], O[16][D]
    static_assert(kDecRows * D * 4 <= kWarpBytes, "a warp's O fits its ring");
};

inline size_t decode_smem(uint32_t ring, uint32_t batch) { return ring + ((size_t)batch + 1) * 8 + 16; }

// The 64-key blocks of a request that some of its new tokens see: the sinks'
// blocks, then those from the first token's window on.
struct Span {
    int32_t lo, sink_end;       // first window key; sinks below it
    uint32_t sink_blocks, first, count;
    __device__ __forceinline__ int32_t key(uint32_t y) const {
        return (int32_t)((y < sink_blocks ? y : first + (y - sink_blocks)) * kDecBlock);
    }
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, const Request& r) {
    Span s;
    s.lo = window_begin(a, r.kv - r.n);
    s.sink_end = (int32_t)min(a.sinks, (uint32_t)s.lo);
    s.sink_blocks = (s.sink_end + kDecBlock - 1) / kDecBlock;
    s.first = max((uint32_t)s.lo / kDecBlock, s.sink_blocks);
    const uint32_t end = ((uint32_t)r.kv + kDecBlock - 1) / kDecBlock;
    // a request without keys still gets its (zero) result from one block
    s.count = max(s.sink_blocks + (end > s.first ? end - s.first : 0u), 1u);
    return s;
}

// This kernel's requests: those whose new tokens and heads fit the 16 rows.
__device__ __forceinline__ bool few_rows(const AttnArgs& a, const Request& r) {
    return r.n > 0 && (uint32_t)r.n <= a.max_q && (uint32_t)r.n * a.group <= kDecRows;
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
            "%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
            "%2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// 16 bytes global -> shared, or 16 zero bytes (nothing is read) where !take.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

// Two adjacent 16-bit values at any 2-byte alignment.
template <typename T>
__device__ __forceinline__ uint32_t load_pair(const T* p) {
    if ((reinterpret_cast<uintptr_t>(p) & 3u) == 0)
        return *reinterpret_cast<const uint32_t*>(p);
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    return (uint32_t)h[0] | ((uint32_t)h[1] << 16);
}

// Four adjacent result values, one store where the address allows it.
template <typename T>
__device__ __forceinline__ void store_out4(const AttnArgs& a, int64_t at, const float (&x)[4]) {
    if (a.out_type == kTypeF32) {
        float* p = reinterpret_cast<float*>(a.out) + at;
        if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
            return;
        }
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + at;
        if ((reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
            *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        store_out<T>(a, at + e, x[e]);
}

template <int D, typename T>
static __global__ void __launch_bounds__(kDecThreads, kDecPerSm) attention_split_kernel(const __grid_constant__ AttnArgs a) {
    using Shape = DecodeShape<D>;
    constexpr uint32_t kStages = Shape::kStages, kStage = Shape::kStageBytes;
    constexpr uint32_t kChunks = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* prefix = reinterpret_cast<uint64_t*>(smem + Shape::kRingBytes);  // [batch + 1] blocks before a request
    __shared__ uint64_t warp_sum[kDecWarps];
    __shared__ float joint_m[kDecWarps][kDecRows], joint_l[kDecWarps][kDecRows];
    __shared__ uint32_t odd_rows;
    __shared__ int last_arriver;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t g = lane >> 2, t4 = lane & 3;  // fragment row and column pair
    griddep_launch_dependents();
    griddep_wait();

    // ---- blocks of every request, and this CTA's share of them
    uint64_t total = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kDecThreads) {
        const uint32_t b = b0 + tid;
        uint64_t x = 0;
        if (b < a.batch) {
            const Request r = load_request(a, b);
            if (r.n > (int32_t)a.max_q && blockIdx.x == 0)
                atomicOr(a.status, kPagedRange);
            x = few_rows(a, r) ? (uint64_t)span_of(a, r).count * a.c.kv_heads : 0;
        }
        uint64_t sum = x;
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, sum, d);
            sum += lane >= d ? y : 0;
        }
        if (lane == 31)
            warp_sum[warp] = sum;
        __syncthreads();
        uint64_t before = total;
#pragma unroll
        for (uint32_t w = 0; w < kDecWarps; ++w) {
            before += w < warp ? warp_sum[w] : 0;
            total += warp_sum[w];
        }
        if (b < a.batch)
            prefix[b] = before + sum - x;
        __syncthreads();
    }
    if (tid == 0)
        prefix[a.batch] = total;
    __syncthreads();
    const uint64_t rows = (uint64_t)a.batch * a.c.kv_heads;
    const uint64_t shares = min((uint64_t)gridDim.x, max((total + kMinShare - 1) / kMinShare, min(rows, total)));
    if (blockIdx.x >= shares)
        return;

    // the request that block x belongs to
    auto request_at = [&](uint64_t x) {
        uint32_t lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (prefix[mid] <= x)
                lo = mid;
            else
                hi = mid;
        }
        return lo;
    };
    // first block of share c: inside a short row it moves to the row's start
    auto share_begin = [&](uint64_t c) {
        const uint64_t x = c * total / shares;
        if (c == 0 || c >= shares)
            return x;
        const uint32_t b = request_at(x);
        const uint64_t len = (prefix[b + 1] - prefix[b]) / a.c.kv_heads;
        return len > kWholeBlocks ? x : x - (x - prefix[b]) % len;
    };
    uint64_t x = share_begin(blockIdx.x);
    const uint64_t x_end = share_begin(blockIdx.x + 1);

    unsigned char* ring = smem + warp * Shape::kWarpBytes;
    const uint32_t ring_addr = smem_addr(ring);
    bool first_segment = true;

    while (x < x_end) {
        // ---- one segment: blocks [y0, y1) of row (b, kvh)
        const uint32_t b = request_at(x);
        const Request r = load_request(a, b);
        const Span sp = span_of(a, r);
        const uint64_t in = x - prefix[b];
        const uint32_t kvh = (uint32_t)(in / sp.count), y0 = (uint32_t)(in % sp.count);
        const uint64_t row_begin = x - y0, row_end = row_begin + sp.count;
        const uint32_t y1 = (uint32_t)(min(x_end, row_end) - row_begin);
        const uint32_t nrows = (uint32_t)r.n * a.group;

        // Q fragments: row i * group + head of the group
        uint32_t qf[D / 16][4];
        int32_t pos[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t row = g + half * 8, i = min(row / a.group, (uint32_t)r.n - 1);
            pos[half] = r.kv - r.n + (int32_t)i;
            lo[half] = window_begin(a, pos[half]);
            const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(r.start + (int32_t)i) * a.q_token +
                         (int64_t)(kvh * a.group + row % a.group) * a.q_head + t4 * 2;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][half] = row < nrows ? load_pair<T>(q + k * 16) : 0u;
                qf[k][half + 2] = row < nrows ? load_pair<T>(q + k * 16 + 8) : 0u;
            }
        }
        float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[n][e] = 0.0f;

        // this warp's tiles: one of each block
        const T* kb = reinterpret_cast<const T*>(a.c.k) + (int64_t)kvh * a.c.k_head;
        const T* vb = reinterpret_cast<const T*>(a.c.v) + (int64_t)kvh * a.c.v_head;
        auto tile_key = [&](uint32_t y) { return sp.key(y) + (int32_t)(warp * kDecTile); };
        auto lookup = [&](uint32_t y) -> int32_t {
            const int32_t j = tile_key(y);
            return y < y1 && j < r.kv ? page_of(a, b, j) : -1;
        };
        // rows that no token sees arrive as zeros: whatever the cache holds
        // there (a weight of zero times NaN is NaN) stays out of the product
        auto fetch = [&](uint32_t y, uint32_t stage, int32_t page) {
            const int32_t j0 = tile_key(y);
            const uint32_t at = ring_addr + stage * kStage;
            const int32_t in_page = j0 & ((1 << a.c.page_shift) - 1);
            const T* kp = kb + (int64_t)max(page, 0) * a.c.k_page;
            const T* vp = vb + (int64_t)max(page, 0) * a.c.v_page;
#pragma unroll
            for (uint32_t i = 0; i < kDecTile * kChunks / 32; ++i) {
                const uint32_t row = i * (32 / kChunks) + lane / kChunks, chunk = lane % kChunks;
                const int32_t j = j0 + (int32_t)row;
                const bool take = page >= 0 && j < r.kv && (j >= sp.lo || j < sp.sink_end);
                const uint32_t dst = at + row * (D * 2) + ((chunk ^ (row & 7u)) * 16u);
                const int64_t off = take ? (int64_t)(in_page + (int32_t)row) : 0;
                copy16(dst, take ? kp + off * a.c.k_row + chunk * 8 : kb, take);
                copy16(dst + kDecTile * D * 2, take ? vp + off * a.c.v_row + chunk * 8 : vb, take);
            }
        };
        int32_t page_ring[kStages];
#pragma unroll
        for (uint32_t s = 0; s < kStages; ++s)
            page_ring[s] = lookup(y0 + s);
#pragma unroll
        for (uint32_t s = 0; s < kStages - 1; ++s) {
            if (y0 + s < y1)
                fetch(y0 + s, s, page_ring[s]);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        for (uint32_t yb = y0; yb < y1; yb += kStages) {
#pragma unroll
            for (uint32_t s = 0; s < kStages; ++s) {
                const uint32_t y = yb + s;
                if (y >= y1)
                    break;
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                __syncwarp();
                const int32_t page = page_ring[s];
                constexpr uint32_t kAhead = kStages - 1;
                const uint32_t sn = (s + kAhead) % kStages;
                if (y + kAhead < y1)
                    fetch(y + kAhead, sn, page_ring[sn]);
                asm volatile("cp.async.commit_group;" ::: "memory");
                page_ring[s] = lookup(y + kStages);

                // S = Q K^T: two 8-key column tiles
                const int32_t j0 = tile_key(y);
                const uint32_t at = ring_addr + s * kStage;
                float sc[2][4] = {};
                {
                    const uint32_t row = (lane & 7u) + ((lane >> 4) & 1u) * 8u;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        uint32_t kf[4];
                        ldmatrix_x4(kf, at + row * (D * 2) + (((k * 2 + ((lane >> 3) & 1u)) ^ (row & 7u)) * 16u));
                        mma_16816<T>(sc[0], qf[k], kf[0], kf[1]);
                        mma_16816<T>(sc[1], qf[k], kf[2], kf[3]);
                    }
                }
                const bool inside = page >= 0 && j0 + (int32_t)kDecTile - 1 <= r.kv - r.n &&
                                    (a.window == 0 || j0 > r.kv - 1 - (int32_t)a.window);
                if (!inside) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int32_t j = j0 + n * 8 + (int32_t)t4 * 2 + (e & 1);
                            const bool seen = page >= 0 && j <= pos[e >> 1] && (j >= lo[e >> 1] || j < (int32_t)a.sinks);
                            sc[n][e] = seen ? sc[n][e] : -INFINITY;
                        }
                }
                // running maximum; O and l move with it
                float mx[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx[h] = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float mn = fmaxf(m[h], mx[h]);
                        const float w = exp2_fast((m[h] - (mn == -INFINITY ? 0.0f : mn)) * a.scale_log2);
                        m[h] = mn;
                        l[h] *= w;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) {
                            o[n][2 * h] *= w;
                            o[n][2 * h + 1] *= w;
                        }
                    }
                }
                uint32_t pf[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float base = m[h] == -INFINITY ? 0.0f : m[h];
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[e] = exp2_fast((sc[e >> 1][2 * h + (e & 1)] - base) * a.scale_log2);
                    l[h] += (p[0] + p[1]) + (p[2] + p[3]);
                    pf[h] = pack2<T>(p[0], p[1]);
                    pf[h + 2] = pack2<T>(p[2], p[3]);
                }
                // O += P V
                {
                    const uint32_t row = (lane & 7u) + ((lane >> 3) & 1u) * 8u;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        uint32_t vf[4];
                        ldmatrix_x4_trans(vf, at + kDecTile * D * 2 + row * (D * 2) +
                                                  (((k * 2 + ((lane >> 4) & 1u)) ^ (row & 7u)) * 16u));
                        mma_16816<T>(o[2 * k], pf, vf[0], vf[1]);
                        mma_16816<T>(o[2 * k + 1], pf, vf[2], vf[3]);
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();

        // ---- the warps' parts: into shared memory, then one sum per value
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (t4 == 0) {
                joint_m[warp][g + 8 * h] = m[h];
                joint_l[warp][g + 8 * h] = l[h];
            }
            float* po = reinterpret_cast<float*>(ring) + (g + 8 * h) * D + t4 * 2;
            if (g + 8 * h < nrows)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
        if (tid == 0)
            odd_rows = 0;
        __syncthreads();

        // shares whose begin lies inside this row: c_lo .. c_hi
        const uint64_t c_lo = row_begin * shares / total + 1;
        uint64_t c_hi = row_end * shares / total;
        while (c_hi >= c_lo && c_hi * total / shares >= row_end)
            --c_hi;
        uint64_t c_first = c_lo;
        while (c_first <= c_hi && c_first * total / shares <= row_begin)
            ++c_first;
        const bool whole = sp.count <= kWholeBlocks || c_first > c_hi;
        const uint32_t parts = whole ? 1u : (uint32_t)(c_hi - c_first + 2);
        // the record of share c's part of a cut row: 1 if the row began in that share, else 0
        float* record = a.partials + (2ull * blockIdx.x + (first_segment && y0 != 0 ? 0u : 1u)) * Shape::kRecord;

        for (uint32_t idx = tid; idx < nrows * (D / 4); idx += kDecThreads) {
            const uint32_t row = idx / (D / 4), d = (idx % (D / 4)) * 4;
            float mm = joint_m[0][row];
#pragma unroll
            for (uint32_t w = 1; w < kDecWarps; ++w)
                mm = fmaxf(mm, joint_m[w][row]);
            const float base = mm == -INFINITY ? 0.0f : mm;
            float v[4] = {}, sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kDecWarps; ++w) {
                const float f = exp2_fast((joint_m[w][row] - base) * a.scale_log2);
                const float4 p = *reinterpret_cast<const float4*>(smem + w * Shape::kWarpBytes + (row * D + d) * 4);
                sum = __fmaf_rn(joint_l[w][row], f, sum);
                v[0] = __fmaf_rn(p.x, f, v[0]);
                v[1] = __fmaf_rn(p.y, f, v[1]);
                v[2] = __fmaf_rn(p.z, f, v[2]);
                v[3] = __fmaf_rn(p.w, f, v[3]);
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = sum == 0.0f ? 0.0f : v[e] * inv;
                    if (!finite32(v[e]))
                        atomicOr(&odd_rows, 1u << row);
                }
                const uint32_t head = kvh * a.group + row % a.group, tok = (uint32_t)r.start + row / a.group;
                store_out4<T>(a, (int64_t)tok * a.o_token + (int64_t)head * a.o_head + d, v);
                if (a.lse && d == 0)
                    a.lse[(int64_t)tok * a.lse_token + head] = sum == 0.0f ? -INFINITY : __fmaf_rn(mm, a.scale, logf(sum));
            } else {
                *reinterpret_cast<float4*>(record + 2 * kDecRows + row * D + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) {
                    record[row] = mm;
                    record[kDecRows + row] = sum;
                }
            }
        }
        if (!whole) {
            // ---- the last of the row's shares to arrive joins all of them
            __threadfence();
            __syncthreads();
            int* counter = a.counters + (uint64_t)b * a.c.kv_heads + kvh;
            if (tid == 0) {
                const int before = atomicAdd(counter, 1);
                last_arriver = before == (int)parts - 1;
                if (last_arriver)
                    *counter = 0;  // as the next call expects it
                __threadfence();
            }
            __syncthreads();
            if (last_arriver) {
                auto part = [&](uint32_t p) {  // in the order of the keys
                    return a.partials + (p == 0 ? 2 * (c_first - 1) + 1 : 2 * (c_first - 1 + p)) * Shape::kRecord;
                };
                float* weight = reinterpret_cast<float*>(smem);  // [parts][nrows]
                for (uint32_t row = warp; row < nrows; row += kDecWarps) {
                    float mm = -INFINITY;
                    for (uint32_t p = lane; p < parts; p += 32)
                        mm = fmaxf(mm, __ldcg(part(p) + row));
#pragma unroll
                    for (int d = 16; d; d >>= 1)
                        mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
                    const float base = mm == -INFINITY ? 0.0f : mm;
                    float sum = 0.0f;
                    for (uint32_t p = lane; p < parts; p += 32) {
                        const float f = exp2_fast((__ldcg(part(p) + row) - base) * a.scale_log2);
                        weight[p * nrows + row] = f;
                        sum = __fmaf_rn(__ldcg(part(p) + kDecRows + row), f, sum);
                    }
#pragma unroll
                    for (int d = 16; d; d >>= 1)
                        sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    if (lane == 0) {
                        joint_l[0][row] = sum;
                        joint_m[0][row] = mm;
                    }
                }
                __syncthreads();
                for (uint32_t idx = tid; idx < nrows * (D / 4); idx += kDecThreads) {
                    const uint32_t row = idx / (D / 4), d = (idx % (D / 4)) * 4;
                    float v[4] = {};
#pragma unroll 8
                    for (uint32_t p = 0; p < parts; ++p) {
                        const float f = weight[p * nrows + row];
                        const float4 q = __ldcg(reinterpret_cast<const float4*>(part(p) + 2 * kDecRows + row * D + d));
                        v[0] = __fmaf_rn(q.x, f, v[0]);
                        v[1] = __fmaf_rn(q.y, f, v[1]);
                        v[2] = __fmaf_rn(q.z, f, v[2]);
                        v[3] = __fmaf_rn(q.w, f, v[3]);
                    }
                    const float sum = joint_l[0][row], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = sum == 0.0f ? 0.0f : v[e] * inv;
                        if (!finite32(v[e]))
                            atomicOr(&odd_rows, 1u << row);
                    }
                    const uint32_t head = kvh * a.group + row % a.group, tok = (uint32_t)r.start + row / a.group;
                    store_out4<T>(a, (int64_t)tok * a.o_token + (int64_t)head * a.o_head + d, v);
                    if (a.lse && d == 0)
                        a.lse[(int64_t)tok * a.lse_token + head] =
                            sum == 0.0f ? -INFINITY : __fmaf_rn(joint_m[0][row], a.scale, logf(sum));
                }
            }
        }
        __syncthreads();
        // a row that came out infinite or NaN may owe it to a value that only
        // later tokens see: again, key by key (one token: every key counts)
        const uint32_t odd = odd_rows;
        if (odd != 0 && r.n > 1)
            for (uint32_t row = warp; row < nrows; row += kDecWarps)
                if (odd >> row & 1u)
                    attention_row<D, T>(a, b, r, (int32_t)(row / a.group), kvh * a.group + row % a.group);
        __syncthreads();
        first_segment = false;
        x = row_begin + y1;
    }
}

}  // namespace paged
}  // namespace bnn
