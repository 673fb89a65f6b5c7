// paged_prefill.cuh - attention of prompt chunks over their pages on the
// 5th-generation tensor cores.
//
// The group's query heads and a request's new tokens are the rows of one
// matrix per KV head (row = token * group + head of the group), cut into
// tiles of 128. For each tile of 128 keys
//   S = Q K^T                     tcgen05.mma, both operands in shared memory
//   P = 2^(c S - c m)             in registers, one thread per row
//   O = O + P V                   tcgen05.mma, P from TMEM, V as it lies (MN-major)
// with a running maximum m and sum l (the online softmax of Milakov and Gimelshein,
// 2018). m moves only when a row's maximum outgrows it by more than 2^kSlack, a
// known refinement; then O (TMEM) and l are scaled by 2^(c (m_old - m_new)). The
// result does not depend on m beyond rounding: weights reach at most 2^kSlack.
// They are rounded to the cache's type, since both operands of a product have one
// type; l sums them unrounded. With 8192 BF16 tokens that rounding takes the
// result's error from 0.0017 of its size, which the exact result's own rounding to
// 16 bits makes, to 0.0022.
//
// A CTA runs one or two such streams; two, so that the tensor core multiplies for one while
// the other's threads take exponentials: two tiles of 128 rows that share the K
// and V tiles (kPair), or, where there are too few rows to fill the GPU, one tile
// of rows whose key tiles the streams take in turn (kTurns), joined at the end as
// the split kernel joins its parts; short caches are one stream's (kSingle).
// Warps: 4 per stream for the softmax (thread = row = TMEM lane), one that issues
// the TMA loads, one that issues the products. K and V arrive page by page
// (one box of up to 128 rows by 64 columns, 128-byte swizzle) in a ring of
// 128-key tiles. A position that no row of the CTA sees may hold anything:
// its scores are replaced, and its V row is overwritten with zeros before
// the product.
//
// Bound: the chain S -> softmax -> P -> products -> S of a tile. Of 3850 clocks
// that a step of 128 keys takes for both row tiles (8192 tokens, 300 us,
// 0.92 PFLOP/s at the 1.7 GHz that the tensor cores leave) a tile's softmax
// works 2450 (exponentials 1420: 128 a row at 16 a clock and SM are 1024) and
// waits 1400 for products and hand-overs; MUFU and tensor pipe are each busy
// half of the time. The TMEM holds S and O of two tiles of 128-wide heads and no
// more, so a third chain, or a second S, has no room. Tried and slower: steps of
// 64 keys with two S buffers (products 64 wide take 53 clocks instead of half of
// 65: 333 us), exponentials on the FMA pipe for a quarter to a half of the
// weights (303 to 316 us: five FMAs of two values cost what they save), weights
// taken with the old maximum (367 us), products in the order in which weights
// arrive (322 us), weights handed over all at once (306 us).
#pragma once

#include <cuda.h>

#include "paged_common.cuh"
#include "paged_decode.cuh"
#include "tcgen05.cuh"

namespace bnn {
namespace paged {

constexpr uint32_t kPfKeys = 128;   // keys of a tile
constexpr uint32_t kPfHalf = 64;    // keys whose weights are handed over at once
constexpr uint32_t kPfRows = 128;   // rows of a tile
constexpr float kSlack = 8.0f;      // log2 of the largest weight

// How a CTA works: one tile of rows; one whose key tiles two streams take in
// turn; two tiles of rows, a stream each.
enum Mode { kSingle, kTurns, kPair };

template <int D, int kMode>
struct PrefillShape {
    static constexpr uint32_t kStreams = kMode == kSingle ? 1 : 2, kQTiles = kMode == kPair ? 2 : 1;
    static constexpr uint32_t kThreads = kStreams * 128 + 64;
    static constexpr uint32_t kTileBytes = kPfKeys * D * 2;  // of K, V or Q
    static constexpr uint32_t kStages = D == 128 ? 5 : 8;
    // 64-wide heads leave TMEM room for P beside S: then Q K^T of the next keys
    // follows as soon as S is in registers, and the softmax need not wait for it
    // (window chunks 198 -> 178 us). 128-wide heads fill the TMEM with S and O, and
    // P takes S's place.
    static constexpr bool kApart = D == 64;
    static constexpr uint32_t kTmemCols = kStreams * 256;
    static_assert(kStreams * (kPfKeys + D + (kApart ? kPfHalf : 0)) <= kTmemCols, "S, O and P of the streams");
    static constexpr uint32_t kBars = 2 * kStages + 6 * kStreams + kQTiles + 1;
    static constexpr size_t kSmem = 1024 + (size_t)(kQTiles + kStages) * kTileBytes + kBars * 8 + 16 * 4 + 64;
    static_assert((D + 2) * kPfRows * 4 <= kStages * kTileBytes, "a stream's O, m and l fit the ring");
};

struct PrefillArgs {
    AttnArgs a;
    CUtensorMap k_map, v_map;
    uint32_t every_request;  // 0: requests of few rows belong to the split kernel
};

// Test hook: n > 0 is a loader that issues the copies of n - 1 tiles and no more,
// so that the waits for the others run out.
static __device__ int g_paged_starve = 0;

// Instruction descriptor: D f32, A and B of one 16-bit type, M = 128; B K-major
// (Q K^T) or MN-major (P V).
template <typename T>
__host__ __device__ constexpr uint32_t f16_idesc(uint32_t n, bool b_mn_major) {
    const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// V's shared-memory descriptor: MN-major, 128-byte swizzle. Eight keys are
// 1024 B apart (SBO); 64 columns on stand kPfKeys * 128 B further (LBO).
__device__ __forceinline__ uint64_t mn_smem_desc(uint32_t saddr) {
    const uint32_t lo = ((saddr >> 4) & 0x3fffu) | ((kPfKeys * 128u >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// True in one thread of the (whole) warp. A tcgen05.mma takes its operands from
// uniform registers: behind this test the compiler knows that one thread runs
// and keeps them there; behind lane == 0 it does not, and each product cost
// some 130 clocks to issue.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Eight adjacent 16-bit values at any 2-byte alignment.
template <typename T>
__device__ __noinline__ uint4 load_row16(const T* p) {
    return make_uint4(load_pair<T>(p), load_pair<T>(p + 2), load_pair<T>(p + 4), load_pair<T>(p + 6));
}

// 32 words to consecutive TMEM columns of this warp's lanes; complete after tmem_wait_st().
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}

// A box of `map` (64 columns from c0, rows from c1 of head c2 of page c3).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1,
                                            int32_t c2, int32_t c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The lowest n bits (none below 1, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Key tiles that rows of tokens at positions p0 .. p1 see.
struct KeyTiles {
    int32_t lo, sink_end, last;  // keys [0, sink_end) and [lo, last]
    uint32_t sink_tiles, first, count;
    __device__ __forceinline__ int32_t key(uint32_t t) const {
        return (int32_t)((t < sink_tiles ? t : first + (t - sink_tiles)) * kPfKeys);
    }
};
__device__ __forceinline__ KeyTiles key_tiles(const AttnArgs& a, int32_t p0, int32_t p1) {
    KeyTiles k;
    k.lo = window_begin(a, p0);
    k.sink_end = (int32_t)min(a.sinks, (uint32_t)k.lo);
    k.last = p1;
    k.sink_tiles = ((uint32_t)k.sink_end + kPfKeys - 1) / kPfKeys;
    k.first = max((uint32_t)k.lo / kPfKeys, k.sink_tiles);
    const uint32_t end = p1 < 0 ? 0u : (uint32_t)p1 / kPfKeys + 1;
    k.count = p1 < 0 ? 0u : k.sink_tiles + (end > k.first ? end - k.first : 0u);
    return k;
}

template <int D, typename T, int kMode>
static __global__ void __launch_bounds__(PrefillShape<D, kMode>::kThreads, 1)
    attention_tiles_kernel(const __grid_constant__ PrefillArgs args) {
    using Shape = PrefillShape<D, kMode>;
    constexpr uint32_t kStreams = Shape::kStreams;
    constexpr uint32_t kStages = Shape::kStages, kTileBytes = Shape::kTileBytes;
    constexpr uint32_t kHalves = D / 64;                // 64-column halves of a tile
    constexpr uint32_t kHalfBytes = kPfKeys * 128;      // 16 KB
    constexpr uint32_t kLoadWarp = kStreams * 4, kMmaWarp = kLoadWarp + 1;
    constexpr uint32_t kQTiles = Shape::kQTiles, kItemRows = kQTiles * kPfRows;
    constexpr bool kApart = Shape::kApart;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(1024) unsigned char pf_smem[];
    const uint32_t raw = smem_addr(pf_smem);
    unsigned char* sm = pf_smem + (((raw + 1023u) & ~1023u) - raw);
    unsigned char* q_sm = sm;
    unsigned char* ring = sm + kQTiles * kTileBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kTileBytes);
    uint64_t* empty = full + kStages;
    uint64_t* q_ready = empty + kStages;   // [kQTiles] Q in shared memory
    uint64_t* s_ready = q_ready + kQTiles;  // [kStreams] a stream's S in TMEM and its last keys' P V done
    uint64_t* p_ready = s_ready + kStreams;        // [kStreams][2] half of its P in TMEM, O scaled
    uint64_t* s_free = p_ready + 2 * kStreams;     // [kStreams] its S in registers (kApart)
    uint64_t* o_ready = s_free + kStreams;         // [kStreams] its P V done (kApart)
    uint64_t* drained = o_ready + kStreams;
    uint32_t* mapped = reinterpret_cast<uint32_t*>(drained + 1);  // [16] bit u: 16-key part u of tile t (mod 16) is in memory
    uint32_t* tmem_slot = mapped + 16;
    __shared__ uint32_t warp_sum[32];
    __shared__ Request found;
    __shared__ uint32_t found_item, found_request;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t t = 0; t < kQTiles; ++t)
            mbar_init(&q_ready[t], kLoadWarp / kQTiles);
        for (uint32_t t = 0; t < kStreams; ++t) {
            mbar_init(&s_ready[t], 1);
            mbar_init(&p_ready[2 * t], 4);
            mbar_init(&p_ready[2 * t + 1], 4);
            mbar_init(&s_free[t], 4);
            mbar_init(&o_ready[t], 1);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
    }
    griddep_wait();

    // ---- which rows: items of kItemRows rows, request by request, heads side by
    // side; the last ones (they see the most keys of a prompt) first
    const uint32_t nth = blockIdx.x / a.c.kv_heads, kvh = blockIdx.x % a.c.kv_heads;
    uint32_t total = 0, x = 0, at = 0;  // a thread's request: its items, those before it
    Request mine = {};
    auto scan = [&](uint32_t b, uint32_t seen) {
        x = 0;
        if (b < a.batch) {
            bool bad;
            mine = load_request(a, b, &bad);
            if (bad || mine.n > (int32_t)a.max_q) {
                if (blockIdx.x == 0)
                    atomicOr(a.status, kPagedRange);
            } else if (mine.n > 0 && (args.every_request || !few_rows(a, mine))) {
                x = ((uint32_t)mine.n * a.group + kItemRows - 1) / kItemRows;
            }
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
        at = seen + sum - x;
        for (uint32_t w = 0; w < Shape::kThreads / 32; ++w) {
            at += w < warp ? warp_sum[w] : 0;
            seen += warp_sum[w];
        }
        return seen;
    };
#pragma unroll 1
    for (uint32_t b0 = 0; b0 < a.batch; b0 += Shape::kThreads) {
        total = scan(b0 + tid, total);
        if (a.batch > Shape::kThreads)
            __syncthreads();
    }
    if (nth >= total)
        return;
    const uint32_t item = total - 1 - nth;
    uint32_t request = tid;
    auto claim = [&]() {
        if (item - at < x) {  // exactly one thread's
            found = mine;
            found_item = item - at;
            found_request = request;
        }
    };
    if (a.batch <= Shape::kThreads) {
        claim();
    } else {
        uint32_t seen = 0;
#pragma unroll 1
        for (request = tid; request - tid < a.batch; request += Shape::kThreads) {
            seen = scan(request, seen);
            claim();
            __syncthreads();
        }
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "r"(Shape::kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t b = found_request;
    const Request r = found;
    const uint32_t row0 = found_item * kItemRows;
    const uint32_t rows = (uint32_t)r.n * a.group;
    const int32_t base_pos = r.kv - r.n;
    const KeyTiles tiles = key_tiles(a, base_pos + (int32_t)(row0 / a.group),
                                     base_pos + (int32_t)(min(row0 + kItemRows, rows) - 1) / (int32_t)a.group);
    const uint32_t count = tiles.count;
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_o = tmem + kStreams * kPfKeys;
    const uint32_t tmem_p = kApart ? tmem_o + kStreams * D : tmem, p_step = kApart ? kPfHalf : kPfKeys;  // a stream's P

    if (warp == kLoadWarp) {
        // ---- K and V tiles, page by page: lane p has the tile's p-th page
        const uint32_t page_rows = min(1u << a.c.page_shift, kPfKeys);
        const uint32_t per_tile = kPfKeys / page_rows;
        constexpr uint32_t kMostPages = kPfKeys / 16;
        uint32_t slot = 0, round = 0;
        const uint32_t fed = min(count, (uint32_t)*reinterpret_cast<volatile int*>(&g_paged_starve) - 1u);  // all of them where it is 0
        // this lane's page of tile t, or -1
        auto lookup = [&](uint32_t t) -> int32_t {
            const int32_t j = tiles.key(t) + (int32_t)(lane * page_rows);
            const bool need = t < count && lane < per_tile && j <= tiles.last && (j + (int32_t)page_rows > tiles.lo || j < tiles.sink_end);
            return need ? page_of(a, b, j) : -1;
        };
        int32_t next = lookup(0);
#pragma unroll 1
        for (uint32_t t = 0; t < fed; ++t) {
            const int32_t page = next;
            next = lookup(t + 1);  // on its way while this tile's copies are issued
            const uint32_t parts = page_rows / 16;
            const uint32_t bits =
                __reduce_or_sync(0xffffffffu, page >= 0 ? ((1u << parts) - 1u) << (lane * parts) : 0u);
            const uint32_t bytes = (uint32_t)__popc(bits) * 16 * D * 2;
            // only a page longer than a tile is entered at another row than its first
            const int32_t in_page = tiles.key(t) & ((1 << a.c.page_shift) - 1);
            int32_t pages[kMostPages];
#pragma unroll
            for (uint32_t p = 0; p < kMostPages; ++p)
                pages[p] = __shfl_sync(0xffffffffu, page, p);
            bool ok = true;
#pragma unroll 1
            for (int which = 0; which < 2; ++which) {
                if (round > 0)
                    ok = warp_wait(&empty[slot], (round - 1) & 1);
                if (!ok)
                    break;
                if (lane == 0) {
                    if (which == 0)
                        mapped[t % 16] = bits;
                    mbar_arrive_expect_tx(&full[slot], bytes);
                }
                __syncwarp();
                // one elected thread issues all copies: issued by a lane each, they
                // took 100 clocks apiece (256 tokens behind 8192 positions in pages of 16:
                // 119 us that way, 93 us this way; 73 us in pages of 64)
                if (elect_one()) {
                    const uint32_t dst = smem_addr(ring + slot * kTileBytes);
                    const CUtensorMap* map = which ? &args.v_map : &args.k_map;
#pragma unroll
                    for (uint32_t p = 0; p < kMostPages; ++p)
                        if (p < per_tile && pages[p] >= 0)
#pragma unroll
                            for (uint32_t h = 0; h < kHalves; ++h)
                                tma_load_4d(dst + p * page_rows * 128 + h * kHalfBytes, map, &full[slot], (int32_t)(h * 64), in_page,
                                            (int32_t)kvh, pages[p]);
                }
                __syncwarp();
                if (++slot == kStages) {
                    slot = 0;
                    ++round;
                }
            }
            if (!ok) {
                if (lane == 0)
                    atomicOr(a.status, kStatusTimeout);
                break;
            }
        }
        // no copy may be in flight when the CTA exits
        const uint32_t issued = round * kStages + slot;
        for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
            if (!wait(&full[i % kStages], (i / kStages) & 1) && lane == 0)
                atomicOr(a.status, kStatusTimeout);
    } else if (warp == kMmaWarp) {
        // ---- the products, all by one thread; Q K^T of the next keys right after P V
        if (elect_one()) {
            constexpr uint32_t kQkDesc = f16_idesc<T>(kPfKeys, false), kPvDesc = f16_idesc<T>(D, true);
            const uint64_t q_desc = mma_smem_desc(smem_addr(q_sm)), k_desc = mma_smem_desc(smem_addr(ring));
            const uint64_t v_desc = mn_smem_desc(smem_addr(ring));
            bool ok = true;
            auto need = [&](uint64_t* bar, uint32_t parity) {
                ok = ok && wait(bar, parity);
                return ok;
            };
            auto slot_of = [&](uint32_t t, uint32_t which) { return (2 * t + which) % kStages; };
            auto parity_of = [&](uint32_t t, uint32_t which) { return ((2 * t + which) / kStages) & 1; };
            auto qk = [&](uint32_t stream, uint32_t t) {
                const uint64_t qa = q_desc + ((kMode == kPair ? stream : 0) * kTileBytes >> 4), ka = k_desc + (slot_of(t, 0) * kTileBytes >> 4);
                const uint32_t to = tmem + stream * kPfKeys;
#pragma unroll
                for (uint32_t k = 0; k < D / 16; ++k) {
                    const uint32_t off = ((k / 4) * kHalfBytes + (k % 4) * 32) >> 4;
                    mma_f16_ss(to, qa + off, ka + off, kQkDesc, k != 0);
                }
            };
            // P V of key tile t, the stream's j-th
            auto pv = [&](uint32_t stream, uint32_t t, uint32_t j) {
                const uint64_t va = v_desc + (slot_of(t, 1) * kTileBytes >> 4);
#pragma unroll 1
                for (uint32_t h = 0; h < 2 && need(&p_ready[2 * stream + h], j & 1); ++h) {
                    tc_fence_after();
#pragma unroll
                    for (uint32_t k = 0; k < kPfHalf / 16; ++k)
                        mma_f16_ts(tmem_o + stream * D, tmem_p + stream * p_step + h * (kPfHalf / 2) + k * 8,
                                   va + ((h * kPfHalf + k * 16) * 128 >> 4), kPvDesc, j != 0 || h != 0 || k != 0);
                }
                return ok;
            };
            if (kMode != kTurns && count > 0 && need(&full[slot_of(0, 0)], 0)) {
#pragma unroll 1
                for (uint32_t stream = 0; stream < kStreams && need(&q_ready[kMode == kPair ? stream : 0], 0); ++stream) {
                    tc_fence_after();
                    qk(stream, 0);
                    mma_commit(&s_ready[stream]);
                }
                mma_commit(&empty[slot_of(0, 0)]);
#pragma unroll 1
                for (uint32_t t = 0; ok && t < count; ++t) {
                    const bool more = t + 1 < count;
                    auto next_scores = [&](uint32_t stream) {
                        if (more && (stream != 0 || need(&full[slot_of(t + 1, 0)], parity_of(t + 1, 0))))
                            qk(stream, t + 1);
                        if (more && stream == kStreams - 1)
                            mma_commit(&empty[slot_of(t + 1, 0)]);
                    };
                    if constexpr (kApart) {
#pragma unroll 1
                        for (uint32_t stream = 0; more && stream < kStreams && need(&s_free[stream], t & 1); ++stream) {
                            tc_fence_after();
                            next_scores(stream);
                            mma_commit(&s_ready[stream]);
                        }
                    }
                    if (!need(&full[slot_of(t, 1)], parity_of(t, 1)))
                        break;
#pragma unroll 1
                    for (uint32_t stream = 0; stream < kStreams && pv(stream, t, t); ++stream) {
                        if constexpr (kApart) {
                            mma_commit(&o_ready[stream]);
                        } else {
                            next_scores(stream);
                            mma_commit(&s_ready[stream]);
                        }
                    }
                    mma_commit(&empty[slot_of(t, 1)]);
                }
            }
            if (kMode == kTurns && count > 0 && need(&q_ready[0], 0)) {
                // scores of key tile t, and its K tile free again
                auto scores = [&](uint32_t t) {
                    if (!need(&full[slot_of(t, 0)], parity_of(t, 0)))
                        return;
                    tc_fence_after();
                    qk(t & 1, t);
                    mma_commit(&empty[slot_of(t, 0)]);
                };
#pragma unroll 1
                for (uint32_t t = 0; t < min(count, 2u); ++t) {
                    scores(t);
                    mma_commit(&s_ready[t]);
                }
#pragma unroll 1
                for (uint32_t t = 0; ok && t < count; ++t) {
                    const uint32_t stream = t & 1, j = t / 2;
                    if (kApart && t + 2 < count && need(&s_free[stream], j & 1)) {
                        scores(t + 2);
                        mma_commit(&s_ready[stream]);
                    }
                    if (!need(&full[slot_of(t, 1)], parity_of(t, 1)) || !pv(stream, t, j))
                        break;
                    if (kApart) {
                        mma_commit(&o_ready[stream]);
                    } else {
                        if (t + 2 < count)
                            scores(t + 2);
                        mma_commit(&s_ready[stream]);
                    }
                    mma_commit(&empty[slot_of(t, 1)]);
                }
            }
            if (!ok)
                atomicOr(a.status, kStatusTimeout);
            // the TMEM may go when every product issued has completed
            mma_commit(drained);
        }
        __syncwarp();
        if (!wait(drained, 0) && lane == 0)
            atomicOr(a.status, kStatusTimeout);
    } else {
        // ---- softmax: thread = row
        const uint32_t stream = warp / 4, wrow = row0 + (kMode == kPair ? stream * kPfRows : 0) + (warp % 4) * 32;  // the warp's first row
        const uint32_t lane_off = ((warp % 4) * 32u) << 16;
        const uint32_t t_s = tmem + stream * kPfKeys + lane_off, t_o = tmem_o + stream * D + lane_off;
        const uint32_t t_p = tmem_p + stream * p_step + lane_off;
        {
            // each warp loads 32 rows of its stream's tile, or 16 of the only one
            constexpr uint32_t kChunks = D / 8, kAtOnce = 32 / kChunks, kLoadRows = kMode == kTurns ? 16 : 32;
            unsigned char* q = q_sm + (kMode == kPair ? stream : 0) * kTileBytes;
            const uint32_t first = kMode == kTurns ? warp * 16 : (warp % 4) * 32;  // in the tile
            const bool q_aligned = ((reinterpret_cast<uintptr_t>(a.q) | (uint64_t)a.q_token * 2 | (uint64_t)a.q_head * 2) & 15u) == 0;
            constexpr uint32_t kLoads = kLoadRows / kAtOnce;
            const uint32_t chunk = lane % kChunks;
            uint32_t row = row0 + (kMode == kPair ? stream * kPfRows : 0) + first + lane / kChunks, tok = row / a.group, head = row % a.group;
            const T* base = reinterpret_cast<const T*>(a.q) + (int64_t)r.start * a.q_token + (int64_t)(kvh * a.group) * a.q_head + chunk * 8;
            uint4 w[kLoads];
            // all of the warp's rows at once, nothing between the loads that would
            // make one wait for another
            if (q_aligned) {
#pragma unroll
                for (uint32_t i = 0; i < kLoads; ++i) {
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (row < rows)
                        w[i] = *reinterpret_cast<const uint4*>(base + (int64_t)tok * a.q_token + (int64_t)head * a.q_head);
                    row += kAtOnce;
                    for (head += kAtOnce; head >= a.group; head -= a.group)
                        ++tok;
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kLoads; ++i) {
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (row < rows)
                        w[i] = load_row16<T>(base + (int64_t)tok * a.q_token + (int64_t)head * a.q_head);
                    row += kAtOnce;
                    for (head += kAtOnce; head >= a.group; head -= a.group)
                        ++tok;
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t tr = first + i * kAtOnce + lane / kChunks;
                *reinterpret_cast<uint4*>(q + (chunk / 8) * kHalfBytes + tr * 128 + (((chunk % 8) ^ (tr & 7u)) * 16u)) = w[i];
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&q_ready[kMode == kPair ? stream : 0]);
        }
        const uint32_t my_row = wrow + lane;
        const int32_t token = (int32_t)min(my_row / a.group, (uint32_t)r.n - 1);
        const int32_t pos = base_pos + token, lo = window_begin(a, pos);
        const int32_t first_pos = base_pos + (int32_t)min(wrow / a.group, (uint32_t)r.n - 1);
        const int32_t last_lo = window_begin(a, base_pos + (int32_t)min((wrow + 31) / a.group, (uint32_t)r.n - 1));
        const float c = a.scale_log2;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        const uint32_t steps = kMode == kTurns ? (count + 1 - stream) / 2 : count;  // this stream's
#pragma unroll 1
        for (uint32_t j = 0; j < steps; ++j) {
            const uint32_t t = kMode == kTurns ? 2 * j + stream : j;  // key tile
            if (!(ok = warp_wait(&s_ready[stream], j & 1)))
                break;
            tc_fence_after();
            uint32_t s[kPfKeys];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                tmem_ld32(t_s + i * 32, s + i * 32);
            const int32_t key0 = tiles.key(t);
            const uint32_t bits = mapped[t % 16];  // written before the K tile's load, which S came after
            if ((kMode == kTurns || stream == 0) && (bits != 0xffu || key0 + (int32_t)kPfKeys - 1 > tiles.last || key0 < tiles.lo)) {
                // V rows that no row of this CTA sees become zeros before the first
                // product with them (which waits for this stream's P)
                const uint32_t slot = (2 * t + 1) % kStages;
                if (!(ok = warp_wait(&full[slot], ((2 * t + 1) / kStages) & 1)))
                    break;
                unsigned char* v = ring + slot * kTileBytes;
#pragma unroll 1
                for (uint32_t row = tid % 128 / 8; row < kPfKeys; row += 16) {
                    const int32_t j = key0 + (int32_t)row;
                    const bool used = (bits >> (row / 16) & 1u) && j <= tiles.last && (j >= tiles.lo || j < tiles.sink_end);
                    if (!used)
#pragma unroll
                        for (uint32_t i = 0; i < kHalves; ++i)
                            *reinterpret_cast<uint4*>(v + i * kHalfBytes + row * 128 + (lane % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async();
            }
            tmem_wait();
            if constexpr (kApart) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&s_free[stream]);
            }
            if (bits != 0xffu || key0 + (int32_t)kPfKeys - 1 > first_pos || (a.window && key0 < last_lo)) {
                // at the edges of what the rows see: hidden scores to -inf
                const int32_t hi = pos - key0, low = lo - key0, sink = (int32_t)a.sinks - key0;
#pragma unroll
                for (int32_t i = 0; i < (int32_t)kPfKeys; i += 32) {
                    const uint32_t parts = bits >> (i / 16);
                    const uint32_t seen = low_bits(hi - i + 1) & (~low_bits(low - i) | low_bits(sink - i)) &
                                          ((parts & 1u ? 0xffffu : 0u) | (parts & 2u ? 0xffff0000u : 0u));
#pragma unroll
                    for (int32_t e = 0; e < 32; ++e)
                        s[i + e] = seen & (1u << e) ? s[i + e] : 0xff800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mx[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 4]));
#pragma unroll
            for (int i = 8; i < (int)kPfKeys; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx[e] = max3(mx[e], __uint_as_float(s[i + e]), __uint_as_float(s[i + e + 4]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool grow = top > m && (top - m) * c > kSlack;  // also the first finite score
            if constexpr (kApart) {
                // the last keys' product has read P and is in O
                if (j > 0 && !(ok = warp_wait(&o_ready[stream], (j - 1) & 1)))
                    break;
                tc_fence_after();
            }
            if (__any_sync(0xffffffffu, grow)) {
                const float mn = grow ? top : m, w = grow ? exp2_fast((m - mn) * c) : 1.0f;
                if (j > 0) {
                    // the product of the last keys has completed (s_ready, o_ready)
#pragma unroll 1
                    for (uint32_t i = 0; i < D / 32; ++i) {
                        uint32_t o[32];
                        tmem_ld32(t_o + i * 32, o);
                        tmem_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * w);
                        tmem_st32(t_o + i * 32, o);
                    }
                }
                l *= w;
                m = mn;
            }
            const float neg = m == -INFINITY ? 0.0f : -m * c;
            const uint64_t c2 = f2_pack(c, c), n2 = f2_pack(neg, neg);
            uint64_t sum2[2] = {0, 0};
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                uint32_t p[32];
#pragma unroll
                for (uint32_t e = 0; e < kPfHalf; e += 2) {
                    const uint32_t i = h * kPfHalf + e;
                    const uint64_t y = f2_fma((uint64_t)s[i] | ((uint64_t)s[i + 1] << 32), c2, n2);
                    const float w0 = exp2_fast(f2_lo(y)), w1 = exp2_fast(f2_hi(y));
                    sum2[(e / 2) & 1] = f2_add(sum2[(e / 2) & 1], f2_pack(w0, w1));
                    p[e / 2] = pack2<T>(w0, w1);
                }
                tmem_st32(t_p + h * (kPfHalf / 2), p);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&p_ready[2 * stream + h]);
            }
            l += (f2_lo(sum2[0]) + f2_hi(sum2[0])) + (f2_lo(sum2[1]) + f2_hi(sum2[1]));
        }
        // every product of stream s is in its O
        auto finished = [&](uint32_t s, uint32_t n) { return n == 0 || (kApart ? warp_wait(&o_ready[s], (n - 1) & 1) : warp_wait(&s_ready[s], n & 1)); };
        ok = ok && finished(stream, steps);
        float* joint = reinterpret_cast<float*>(ring);  // stream 1's O [column][row], then m and l
        if (kMode == kTurns) {
            if (stream == 1) {
                ok = ok && finished(0, (count + 1) / 2);  // then the ring is free
                tc_fence_after();
                const uint32_t row = tid % 128;
                if (ok) {
#pragma unroll 1
                    for (uint32_t i = 0; steps > 0 && i < D / 32; ++i) {
                        uint32_t o[32];
                        tmem_ld32(t_o + i * 32, o);
                        tmem_wait();
#pragma unroll
                        for (uint32_t e = 0; e < 32; ++e)
                            joint[(i * 32 + e) * kPfRows + row] = __uint_as_float(o[e]);
                    }
                    joint[D * kPfRows + row] = m;
                    joint[(D + 1) * kPfRows + row] = l;
                }
            }
            named_barrier(1, 256);
        }
        if (!ok && lane == 0)
            atomicOr(a.status, kStatusTimeout);
        if (ok && (kMode != kTurns || stream == 0)) {
            tc_fence_after();
            float w0 = 1.0f, w1 = 0.0f;  // of the streams' O
            if (kMode == kTurns && count > 1) {
                const uint32_t row = tid % 128;
                const float m1 = joint[D * kPfRows + row], l1 = joint[(D + 1) * kPfRows + row];
                const float both = fmaxf(m, m1), from = both == -INFINITY ? 0.0f : both;
                w0 = exp2_fast((m - from) * c);
                w1 = exp2_fast((m1 - from) * c);
                m = both;
                l = __fmaf_rn(l, w0, l1 * w1);
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const uint32_t head = kvh * a.group + my_row % a.group;
            const int64_t tok = r.start + (int64_t)(my_row / a.group);
            const int64_t at = tok * a.o_token + (int64_t)head * a.o_head;
            bool odd = false;
            unsigned char* to = a.out + at * 2;
            const bool wide = a.out_type != kTypeF32 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
#pragma unroll 1
            for (uint32_t i = 0; i < D / 32; ++i) {
                uint32_t o[32];
                float x[32];
                if (count > 0) {
                    tmem_ld32(t_o + i * 32, o);
                    tmem_wait();
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float v = __uint_as_float(o[e]);
                    if (kMode == kTurns && count > 1)
                        v = __fmaf_rn(joint[(i * 32 + e) * kPfRows + tid % 128], w1, v * w0);
                    x[e] = l == 0.0f ? 0.0f : v * inv;
                    odd |= !finite32(x[e]);
                }
                if (my_row < rows && wide) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(to + (i * 32 + e) * 2) =
                            make_uint4(pack2<T>(x[e], x[e + 1]), pack2<T>(x[e + 2], x[e + 3]), pack2<T>(x[e + 4], x[e + 5]),
                                       pack2<T>(x[e + 6], x[e + 7]));
                } else if (my_row < rows) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        store_out4_any<T>(a, at + i * 32 + e, x[e], x[e + 1], x[e + 2], x[e + 3]);
                }
                __syncwarp();
            }
            odd = odd && my_row < rows && !isnan(l);  // a sum that is no number: the row sees such a score
            if (a.lse && my_row < rows)
                a.lse[tok * a.lse_token + head] = l == 0.0f ? -INFINITY : __fmaf_rn(m, a.scale, ln_fast(l));
            // a row that came out infinite or NaN may owe it to a value that
            // only other tokens see, or in BF16 to weights above one
            uint32_t again = __ballot_sync(0xffffffffu, odd);
            __syncwarp();  // the results are read back
            while (again) {
                const uint32_t i = (uint32_t)__ffs((int)again) - 1;
                again &= again - 1;
                attention_row<D, T, !std::is_same<T, __half>::value>(a, b, r, (int32_t)((wrow + i) / a.group),
                                                                     kvh * a.group + (wrow + i) % a.group, tiles.lo, tiles.last);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kTmemCols));
    }
}

}  // namespace paged
}  // namespace bnn
