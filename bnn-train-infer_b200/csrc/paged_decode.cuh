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
// 16-key tiles through a ring of cp.async stages, across the rows of its share:
// the next row's tiles are on their way while the warps' parts of this one are
// joined. The code is kept small on purpose: a short call runs most of it
// once, and its instructions come from memory.
#pragma once

#include <type_traits>

#include "paged_common.cuh"

namespace bnn {
namespace paged {

// Measured on a B200 (copy rate 6.54 TB/s): 2 requests of 131071 positions,
// 1.07 GB, 167 us = 6.4 TB/s; 8 of 4096 29.4 us, of which 5 us pass until the
// first keys are in (lengths, then page numbers, then keys: three dependent
// reads) and 4 us in the joins; 61 of 1 to 16384 75 us; one of 160 8 us.
constexpr uint32_t kDecWarps = 4;
constexpr uint32_t kDecThreads = kDecWarps * 32;
constexpr uint32_t kDecTile = 16;                     // keys of a warp's step
constexpr uint32_t kDecBlock = kDecTile * kDecWarps;  // keys of a CTA's step
constexpr uint32_t kDecPerSm = 2;                     // CTAs an SM holds: 192 KB of ring
// Rows of this many blocks are not cut: a join costs about as much as they do. With
// 4, 8 and 16: one request of 600 positions (8 KV heads) 10.3, 10.3 and 14.7 us,
// 32 of 300 13.4, 10.8 and 10.8, 32 of 600 18.7, 18.8 and 16.1, 61 ragged ones of
// up to 3000 57.6, 58.4 and 64.5.
constexpr uint32_t kWholeBlocks = 8;
// Units (below) of a share at least. With 2, 4 and 8: one request of 600 positions
// 8.8, 10.2 and 13.4 us, of 4000 11.6, 13.3 and 15.5, 8 of 600 10.3, 11.4 and
// 14.8, 8 of 1000 12.1, 12.1 and 15.5; longer calls are alike.
constexpr uint32_t kMinShare = 4;
// A row's fixed work (its queries, the pipeline's start, the joint sum) in
// units of the time a block takes: shares are equal in blocks plus rows (61
// ragged requests: 132 us with 0, 78 with 2, 73 with 3 on the same code).
constexpr uint32_t kRowCost = 3;
constexpr uint32_t kDecRows = 16;
constexpr uint32_t kLongCache = 2048;   // positions
constexpr uint32_t kSplitGroups = 128;  // groups of 16 rows in a call (all requests and KV heads)
constexpr uint32_t kJoin = 16;          // parts of a row that one CTA joins at a time

template <int D>
struct DecodeShape {
    static constexpr uint32_t kStageBytes = 2 * kDecTile * D * 2;  // K and V rows of a tile
    static constexpr uint32_t kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kWarpBytes = kStages * kStageBytes;
    static constexpr uint32_t kRingBytes = kDecWarps * kWarpBytes;
    static constexpr uint32_t kRecord = kDecRows * (D + 2);  // floats of a partial: m[16], l[16], O[16][D]
    static_assert(kDecRows * D * 4 <= kStageBytes, "a warp's O fits a stage");
};

// The ring, then the requests. From some 1000 requests on (16 bytes each) only one
// CTA fits an SM: 1000 requests of 500 positions run at 4.3 TB/s, 1100 at 3.1.
inline size_t decode_smem(uint32_t ring, uint32_t batch) { return ring + ((size_t)batch + 1) * (4 + sizeof(Request)); }

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

// This kernel's requests: those whose new tokens and heads fit the 16 rows, and
// those behind a long cache whose rows make few enough groups of 16 (each group
// reads the cache again, from L2 mostly). A tile's keys stay on one SM, here
// they spread over all. 8 KV heads, group 2, pages of 16, tiles against groups:
// behind 8192 positions 92 us for up to 128 rows against 30 (24 tokens), 69 (100
// tokens, 104 groups) and 114 us (200 tokens); two requests of 64 behind 4000
// about the same (128 groups, 52 us), four 57 and 83 us; 100 behind 1000 20 and
// 25 us.
__device__ __forceinline__ bool few_rows(const AttnArgs& a, const Request& r) {
    const uint32_t rows = (uint32_t)r.n * a.group;
    return r.n > 0 && (uint32_t)r.n <= a.max_q &&
           (a.split_all || rows <= kDecRows || (rows <= a.split_rows && r.kv >= (int32_t)kLongCache));
}
__device__ __forceinline__ uint32_t row_groups(const AttnArgs& a, const Request& r) {
    return ((uint32_t)r.n * a.group + kDecRows - 1) / kDecRows;
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

// Four adjacent result values at any alignment and of either type.
template <typename T>
__device__ __noinline__ void store_out4_any(const AttnArgs& a, int64_t at, float x0, float x1, float x2, float x3) {
    store_out<T>(a, at, x0);
    store_out<T>(a, at + 1, x1);
    store_out<T>(a, at + 2, x2);
    store_out<T>(a, at + 3, x3);
}
template <typename T>
__device__ __forceinline__ void store_out4(const AttnArgs& a, int64_t at, const float (&x)[4]) {
    uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + at;
    if (a.out_type != kTypeF32 && (reinterpret_cast<uintptr_t>(p) & 7u) == 0)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    else
        store_out4_any<T>(a, at, x[0], x[1], x[2], x[3]);
}

// Counts this CTA in: what its threads wrote before the barrier ahead of this
// is visible to whoever counts last, and theirs to it.
__device__ __forceinline__ int arrive(int* counter) {
    int before;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

// One stretch of a share: blocks [y0, y1) of row (b, kvh, group of 16 of the
// matrix's rows from `first` on). The row's units begin at row_begin, kRowCost
// of them before those of its blocks.
struct Segment {
    Request r;
    Span sp;
    uint32_t b, kvh, first, row_begin, y0, y1;
    __device__ __forceinline__ uint32_t row_end() const { return row_begin + kRowCost + sp.count; }
    __device__ __forceinline__ uint32_t next() const { return row_begin + kRowCost + y1; }  // where its successor begins
};

// Scales and writes four values of one output row (and its lse with d == 0);
// notes a row that is not finite although its sum is a number (a score that is
// none is one that the row sees).
template <typename T>
__device__ __noinline__ void finish4(const AttnArgs& a, const Segment& s, uint32_t in_group, uint32_t d, float4 p, float sum, float mm,
                                     uint32_t* odd_rows, uint32_t bit) {
    const uint32_t row = s.first + in_group, tok = (uint32_t)s.r.start + row / a.group, head = s.kvh * a.group + row % a.group;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float v[4] = {p.x * inv, p.y * inv, p.z * inv, p.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = sum == 0.0f ? 0.0f : v[e];
        if (!finite32(v[e]) && !isnan(sum))
            atomicOr(odd_rows, 1u << bit);
    }
    store_out4<T>(a, (int64_t)tok * a.o_token + (int64_t)head * a.o_head + d, v);
    if (a.lse && d == 0)
        a.lse[(int64_t)tok * a.lse_token + head] = sum == 0.0f ? -INFINITY : __fmaf_rn(mm, a.scale, ln_fast(sum));
}

// A row of which this CTA's share has a part: its shares c_first - 1 .. and so on.
struct Cut {
    Segment s;
    uint32_t c_first, parts, first_of_group, n;
    bool joins_group;
    // where the p-th part, or the group that begins with it, has its record: a
    // share ends one cut row (0) and begins another (1) at most
    __device__ __forceinline__ uint32_t place(uint32_t p) const { return 2 * (c_first - 1 + p) + (p == 0 ? 1u : 0u); }
};

template <int D, typename T>
static __global__ void __launch_bounds__(kDecThreads, kDecPerSm) attention_split_kernel(const __grid_constant__ AttnArgs a) {
    using Shape = DecodeShape<D>;
    constexpr uint32_t kStages = Shape::kStages, kStage = Shape::kStageBytes;
    constexpr uint32_t kChunks = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(128) unsigned char smem[];
    uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + Shape::kRingBytes);  // [batch + 1] units before a request
    Request* requests = reinterpret_cast<Request*>(prefix + a.batch + 1);
    __shared__ uint32_t warp_sum[kDecWarps];
    __shared__ float joint_m[kDecWarps][kDecRows], joint_l[kDecWarps][kDecRows];
    __shared__ uint32_t odd_rows;
    __shared__ Cut cut[2];

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t g = lane >> 2, t4 = lane & 3;  // fragment row and column pair
    griddep_launch_dependents();
    griddep_wait();

    // ---- what every request costs, in units (kRowCost and one for each block of
    // a row), and this CTA's share of it
    uint32_t total = 0;
#pragma unroll 1
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kDecThreads) {
        const uint32_t b = b0 + tid;
        uint32_t x = 0;
        if (b < a.batch) {
            bool bad;
            const Request r = load_request(a, b, &bad);
            requests[b] = r;
            if ((bad || r.n > (int32_t)a.max_q) && blockIdx.x == 0)
                atomicOr(a.status, kPagedRange);
            x = few_rows(a, r) ? (span_of(a, r).count + kRowCost) * a.c.kv_heads * row_groups(a, r) : 0;
        }
        uint32_t sum = x;
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, sum, d);
            sum += lane >= d ? y : 0;
        }
        if (lane == 31)
            warp_sum[warp] = sum;
        __syncthreads();
        uint32_t before = total;
#pragma unroll
        for (uint32_t w = 0; w < kDecWarps; ++w) {
            before += w < warp ? warp_sum[w] : 0;
            total += warp_sum[w];
        }
        if (b < a.batch)
            prefix[b] = before + sum - x;
        __syncthreads();
    }
    if (tid == 0) {
        prefix[a.batch] = total;
        odd_rows = 0;
    }
    __syncthreads();
    if (total == 0)
        return;
    const uint32_t rows = a.batch * a.c.kv_heads;
    const uint32_t shares = min(gridDim.x, max((total + kMinShare - 1) / kMinShare, min(rows, total)));
    if (blockIdx.x >= shares)
        return;
    const uint32_t even = total / shares, extra = total % shares;  // the first `extra` shares have one unit more

    // the request that unit x belongs to (all lanes of a warp ask for the same x:
    // 32 prefixes a look)
    uint32_t widest = 1;
    while (widest * 32 < a.batch)
        widest *= 32;
    auto request_at = [&](uint32_t x) {
        uint32_t lo = 0;
#pragma unroll 1
        for (uint32_t step = widest; step; step /= 32) {
            const uint32_t b = lo + lane * step;
            lo += (__popc(__ballot_sync(0xffffffffu, b < a.batch && prefix[b] <= x)) - 1) * step;
        }
        return lo;
    };
    // first unit of share c; inside a short row, or before a row's first block,
    // it moves to the row's start
    auto raw_begin = [&](uint32_t c) { return c * even + min(c, extra); };
    uint32_t ends[2];
#pragma unroll 1
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t at = raw_begin(blockIdx.x + i);
        uint32_t begin = at;
        if (at < total) {
            const uint32_t b = request_at(at), len = span_of(a, requests[b]).count + kRowCost, in = (at - prefix[b]) % len;
            begin = len > kWholeBlocks + kRowCost && in > kRowCost ? at : at - in;
        }
        ends[0] = i == 0 ? begin : ends[0];
        ends[1] = begin;
    }
    const uint32_t x_begin = ends[0], x_end = ends[1];
    if (x_begin >= x_end)
        return;
    auto segment_at = [&](uint32_t x) {
        Segment s;
        s.b = request_at(x);
        s.r = requests[s.b];
        s.sp = span_of(a, s.r);
        const uint32_t in = x - prefix[s.b], len = s.sp.count + kRowCost;
        const uint32_t nth = in / len, groups = row_groups(a, s.r);
        s.kvh = nth / groups;
        s.first = (nth - s.kvh * groups) * kDecRows;
        const uint32_t y = in - nth * len;
        s.row_begin = x - y;
        s.y0 = y > kRowCost ? y - kRowCost : 0;
        s.y1 = min(x_end - s.row_begin, len) - kRowCost;
        return s;
    };

    const uint32_t ring_addr = smem_addr(smem) + warp * Shape::kWarpBytes;
    const uint32_t page_mask = (1u << a.c.page_shift) - 1u;
    auto tile_key = [&](const Segment& s, uint32_t y) { return s.sp.key(y) + (int32_t)(warp * kDecTile); };

    // ---- what is fetched: the next tile is block fy of segment f, whose units
    // begin at fx; the lanes hold the pages of its 32 blocks from `base` on, and of
    // the 32 after them
    Segment f = segment_at(x_begin);
    uint32_t fx = x_begin, fy = f.y0, base = fy, slot_f = 0;
    auto lookup = [&](uint32_t y) -> int32_t {
        if (y >= f.y1)
            return -1;
        const int32_t j = tile_key(f, y);
        return j < f.r.kv ? page_of(a, f.b, j) : -1;
    };
    int32_t pages = lookup(base + lane), more = -1;
    uint32_t valid = 0, in_flight = 0;  // bit i: the i-th tile in flight lies in a page
    // rows that no token sees arrive as zeros: whatever the cache holds
    // there (a weight of zero times NaN is NaN) stays out of the product
    auto fetch = [&]() {
        if (fx < x_end) {
            const int32_t page = __shfl_sync(0xffffffffu, pages, (int)(fy - base));
            const int32_t j0 = tile_key(f, fy);
            const uint32_t at = ring_addr + slot_f * kStage;
            const int64_t head = (int64_t)f.kvh, in_page = (int64_t)((uint32_t)j0 & page_mask);
            const T* kp = reinterpret_cast<const T*>(a.c.k);
            const T* vp = reinterpret_cast<const T*>(a.c.v);
            if (page >= 0) {
                kp += head * a.c.k_head + (int64_t)page * a.c.k_page + in_page * a.c.k_row;
                vp += head * a.c.v_head + (int64_t)page * a.c.v_page + in_page * a.c.v_row;
            }
#pragma unroll
            for (uint32_t i = 0; i < kDecTile * kChunks / 32; ++i) {
                const uint32_t row = i * (32 / kChunks) + lane / kChunks, chunk = lane % kChunks;
                const int32_t j = j0 + (int32_t)row;
                const bool take = page >= 0 && j < f.r.kv && (j >= f.sp.lo || j < f.sp.sink_end);
                const uint32_t dst = at + row * (D * 2) + ((chunk ^ (row & 7u)) * 16u);
                copy16(dst, kp + (take ? (int64_t)row * a.c.k_row + chunk * 8 : 0), take);
                copy16(dst + kDecTile * D * 2, vp + (take ? (int64_t)row * a.c.v_row + chunk * 8 : 0), take);
            }
            valid |= (page >= 0 ? 1u : 0u) << in_flight;
            ++in_flight;
            slot_f = slot_f + 1 == kStages ? 0 : slot_f + 1;
            ++fy;
            if (fy == f.y1) {
                fx = f.next();
                if (fx < x_end) {
                    f = segment_at(fx);
                    fy = base = f.y0;
                    pages = lookup(base + lane);
                }
            } else if (fy - base == 32) {
                base = fy;
                pages = more;
            } else if (fy - base == 8) {
                more = lookup(base + 32 + lane);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (uint32_t s = 0; s < kStages - 1; ++s)
        fetch();

    // a row that came out infinite or NaN may owe it to a value that only other
    // tokens see (attention_row)
    // (`first_bit`: where this row's 16 bits of odd_rows begin; two cut rows are
    // noted before either is computed again)
    auto redo = [&](const Segment& s, uint32_t first_bit) {
        __syncthreads();
        if (const uint32_t odd = odd_rows >> first_bit & 0xffffu) {
#pragma unroll 1
            for (uint32_t row = warp; row < kDecRows; row += kDecWarps)
                if (odd >> row & 1u)
                    attention_row<D, T, false>(a, s.b, s.r, (int32_t)((s.first + row) / a.group),
                                               s.kvh * a.group + (s.first + row) % a.group, s.sp.lo, s.r.kv - 1);
            __syncthreads();
            if (tid == 0)
                odd_rows &= ~(0xffffu << first_bit);
            __syncthreads();
        }
    };
    // the share whose stretch of units holds `at`
    auto share_of = [&](uint32_t at) {
        const uint32_t cut = extra * (even + 1);
        return at < cut ? at / (even + 1) : extra + (at - cut) / even;
    };

    uint32_t x = x_begin, slot = 0, cuts = 0;
    bool grouped = false;  // one of the cut rows has more than kJoin parts
    while (x < x_end) {
        // ---- one segment
        const Segment s = segment_at(x);
        const uint32_t nrows = min((uint32_t)s.r.n * a.group - s.first, kDecRows);
        // Q fragments: row i * group + head of the group
        uint32_t qf[D / 16][4];
        int32_t pos[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t row = s.first + g + half * 8, i = min(row / a.group, (uint32_t)s.r.n - 1);
            pos[half] = s.r.kv - s.r.n + (int32_t)i;
            lo[half] = window_begin(a, pos[half]);
            const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(s.r.start + (int32_t)i) * a.q_token +
                         (int64_t)(s.kvh * a.group + row % a.group) * a.q_head + t4 * 2;
            const bool there = g + half * 8 < nrows;
            if ((reinterpret_cast<uintptr_t>(q) & 3u) == 0) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qf[k][half] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16) : 0u;
                    qf[k][half + 2] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) : 0u;
                }
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qf[k][half] = there ? (uint32_t)h[k * 16] | (uint32_t)h[k * 16 + 1] << 16 : 0u;
                    qf[k][half + 2] = there ? (uint32_t)h[k * 16 + 8] | (uint32_t)h[k * 16 + 9] << 16 : 0u;
                }
            }
        }
        const int32_t first_pos = s.r.kv - s.r.n + (int32_t)(s.first / a.group);
        const int32_t last_lo = window_begin(a, s.r.kv - s.r.n + (int32_t)((s.first + nrows - 1) / a.group));
        float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[n][e] = 0.0f;

        uint32_t used = 0;  // the slot of the last tile
#pragma unroll 1
        for (uint32_t y = s.y0; y < s.y1; ++y) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            fetch();
            const bool there = valid & 1u;
            valid >>= 1;
            --in_flight;

            // S = Q K^T: two 8-key column tiles
            const int32_t j0 = tile_key(s, y);
            const uint32_t at = ring_addr + slot * kStage;
            used = slot;
            slot = slot + 1 == kStages ? 0 : slot + 1;
            float sc[2][4] = {};
            {
                float odd[2][4] = {};  // the odd steps apart: half the chain of dependent products
                const uint32_t row = (lane & 7u) + ((lane >> 4) & 1u) * 8u;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t kf[4];
                    ldmatrix_x4(kf, at + row * (D * 2) + (((k * 2 + ((lane >> 3) & 1u)) ^ (row & 7u)) * 16u));
                    mma_16816<T>(k & 1 ? odd[0] : sc[0], qf[k], kf[0], kf[1]);
                    mma_16816<T>(k & 1 ? odd[1] : sc[1], qf[k], kf[2], kf[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[0][e] += odd[0][e];
                    sc[1][e] += odd[1][e];
                }
            }
            const bool inside = there && j0 + (int32_t)kDecTile - 1 <= first_pos && (a.window == 0 || j0 >= last_lo);
            if (!inside) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t j = j0 + n * 8 + (int32_t)t4 * 2 + (e & 1);
                        const bool seen = there && j <= pos[e >> 1] && (j >= lo[e >> 1] || j < (int32_t)a.sinks);
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
            // The weights are rounded to the cache's type: both operands of a product have
            // one. The sum keeps them unrounded, so that it brings no rounding of its own
            // into the result and lse. An F16 weight below 2^-25 of the row's largest so
            // far is lost to the product.
            uint32_t pf[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float from = m[h] == -INFINITY ? 0.0f : m[h];
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p[e] = exp2_fast((sc[e >> 1][2 * h + (e & 1)] - from) * a.scale_log2);
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

        // ---- the warps' parts: into the slots of the last tile (free until the
        // next one is fetched), then one sum per value
        __syncwarp();
        unsigned char* part_o = smem + used * kStage;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (t4 == 0) {
                joint_m[warp][g + 8 * h] = m[h];
                joint_l[warp][g + 8 * h] = l[h];
            }
            float* po = reinterpret_cast<float*>(part_o + warp * Shape::kWarpBytes) + (g + 8 * h) * D + t4 * 2;
            if (g + 8 * h < nrows)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
        __syncthreads();

        // shares that begin behind this row's first block: c_first .. c_last
        const uint32_t c_first = share_of(s.row_begin + kRowCost) + 1, c_last = share_of(s.row_end() - 1);
        const bool whole = s.sp.count <= kWholeBlocks || c_first > c_last;
        if (!whole && tid == 0) {
            // at most two: the row that an earlier share began, and the last one
            Cut& k = cut[cuts];
            k.s = s;
            k.c_first = c_first;
            k.parts = c_last - c_first + 2;
            k.first_of_group = (blockIdx.x - (c_first - 1)) / kJoin * kJoin;
            k.joins_group = false;
        }
        // the record of this share's part of a cut row: 1 if the row begins in this share, else 0
        float* record = a.partials + (2ull * blockIdx.x + (s.y0 != 0 ? 0u : 1u)) * Shape::kRecord;

#pragma unroll 1
        for (uint32_t idx = tid; idx < nrows * (D / 4); idx += kDecThreads) {
            const uint32_t row = idx / (D / 4), d = (idx % (D / 4)) * 4;
            float mm = joint_m[0][row];
#pragma unroll
            for (uint32_t w = 1; w < kDecWarps; ++w)
                mm = fmaxf(mm, joint_m[w][row]);
            const float from = mm == -INFINITY ? 0.0f : mm;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kDecWarps; ++w) {
                const float e = exp2_fast((joint_m[w][row] - from) * a.scale_log2);
                const float4 p = *reinterpret_cast<const float4*>(part_o + w * Shape::kWarpBytes + (row * D + d) * 4);
                sum = __fmaf_rn(joint_l[w][row], e, sum);
                v.x = __fmaf_rn(p.x, e, v.x);
                v.y = __fmaf_rn(p.y, e, v.y);
                v.z = __fmaf_rn(p.z, e, v.z);
                v.w = __fmaf_rn(p.w, e, v.w);
            }
            if (whole) {
                finish4<T>(a, s, row, d, v, sum, mm, &odd_rows, row);
            } else {
                *reinterpret_cast<float4*>(record + 2 * kDecRows + row * D + d) = v;
                if (d == 0) {
                    record[row] = mm;
                    record[kDecRows + row] = sum;
                }
            }
        }
        if (whole) {
            redo(s, 0);
        } else {
            ++cuts;
            grouped |= c_last - c_first + 2 > kJoin;
            __syncthreads();
        }
        x = s.next();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- cut rows: the last of a row's shares to arrive joins all of them, in
    // the order of the keys; more than kJoin parts first in groups of kJoin (one
    // CTA reading hundreds of parts would take longer than the row). A share
    // arrives when all its work is done: the joint sums hold up no stream.
    if (cuts == 0)
        return;
#pragma unroll 1
    for (uint32_t round = grouped ? 0 : 1; round < 2; ++round) {
        __syncthreads();  // the CTA's records are written
        if (tid < cuts) {
            Cut& k = cut[tid];
            const bool in_groups = k.parts > kJoin;
            k.n = 0;
            if (round == 0 ? in_groups : !in_groups || k.joins_group) {
                const uint32_t n = round == 0 ? min(kJoin, k.parts - k.first_of_group)
                                   : in_groups ? (k.parts + kJoin - 1) / kJoin : k.parts;
                int* counter = round == 0 ? a.group_counters + k.place(k.first_of_group) : a.row_counters + k.place(0);
                if (arrive(counter) == (int)n - 1) {
                    *counter = 0;  // as the next call expects it
                    k.n = n;
                    k.joins_group = round == 0;  // this CTA has joined the group and counts for it
                }
            }
        }
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = 0; i < cuts; ++i) {
            const Cut& k = cut[i];
            const uint32_t n = k.n, nrows = min((uint32_t)k.s.r.n * a.group - k.s.first, kDecRows);
            if (n == 0)
                continue;
            // record of the p-th of the n parts; the groups' lie behind the shares'
            const bool of_groups = round == 1 && k.parts > kJoin;
            const uint32_t p_begin = round == 0 ? k.first_of_group : 0, p_step = of_groups ? kJoin : 1;
            const float* records = a.partials + (of_groups ? 2ull * gridDim.x * Shape::kRecord : 0ull);
            float* joined = a.partials + (2ull * gridDim.x + k.place(k.first_of_group)) * Shape::kRecord;
            // both rows at once where there are two and threads for them
            const uint32_t quads = nrows * (D / 4);
            const uint32_t turn = cuts == 2 && i == 1 && quads <= kDecThreads / 2 ? tid ^ (kDecThreads / 2) : tid;
#pragma unroll 1
            for (uint32_t idx = turn; idx < quads; idx += kDecThreads) {
                const uint32_t row = idx / (D / 4), d = (idx % (D / 4)) * 4;
                float mm = -INFINITY, sum = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                for (uint32_t p0 = 0; p0 < n; p0 += 8) {  // eight parts at once: their loads overlap
                    float pm[8], pl[8];
                    float4 q[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const bool there = p0 + e < n;
                        const float* from = records + (uint64_t)k.place(p_begin + (there ? p0 + e : 0) * p_step) * Shape::kRecord;
                        pm[e] = there ? __ldcg(from + row) : -INFINITY;
                        pl[e] = there ? __ldcg(from + kDecRows + row) : 0.0f;
                        q[e] = there ? __ldcg(reinterpret_cast<const float4*>(from + 2 * kDecRows + row * D + d))
                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                    float to = mm;
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e)
                        to = fmaxf(to, pm[e]);
                    const float base = to == -INFINITY ? 0.0f : to, w = exp2_fast((mm - base) * a.scale_log2);
                    mm = to;
                    sum *= w;
                    v = make_float4(v.x * w, v.y * w, v.z * w, v.w * w);
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const float f = exp2_fast((pm[e] - base) * a.scale_log2);
                        sum = __fmaf_rn(pl[e], f, sum);
                        v.x = __fmaf_rn(q[e].x, f, v.x);
                        v.y = __fmaf_rn(q[e].y, f, v.y);
                        v.z = __fmaf_rn(q[e].z, f, v.z);
                        v.w = __fmaf_rn(q[e].w, f, v.w);
                    }
                }
                if (round == 1) {
                    finish4<T>(a, k.s, row, d, v, sum, mm, &odd_rows, row + kDecRows * i);
                } else {
                    *reinterpret_cast<float4*>(joined + 2 * kDecRows + row * D + d) = v;
                    if (d == 0) {
                        joined[row] = mm;
                        joined[kDecRows + row] = sum;
                    }
                }
            }
        }
    }
#pragma unroll 1
    for (uint32_t i = 0; i < cuts; ++i)
        redo(cut[i].s, kDecRows * i);
}

}  // namespace paged
}  // namespace bnn
