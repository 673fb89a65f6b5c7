// paged.cu - host side of the paged-cache operators (include/bnn_b200_paged.h):
// argument checks, the choice of kernel, launches.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "bnn_b200_paged.h"
#include "bnn_internal.h"
#include "paged_append.cuh"
#include "paged_common.cuh"
#include "paged_decode.cuh"
#include "paged_prefill.cuh"

namespace {

using namespace bnn::paged;

constexpr int64_t kMaxCount = (int64_t)1 << 30;  // tokens, positions, slots

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

BNN_Status check_cache(const BNN_PagedCache& c, Cache* out) {
    if (c.type != BNN_PAGED_BF16 && c.type != BNN_PAGED_F16)
        return BNN_EINVAL;
    if (c.head_dim != 64 && c.head_dim != 128)
        return BNN_ENOTSUP;
    uint32_t shift = 0;
    for (; shift <= 8 && c.page_size != ((int64_t)1 << shift); ++shift) {
    }
    if (shift < 4 || shift > 8)
        return BNN_ENOTSUP;
    if (c.kv_heads <= 0 || c.kv_heads > 65536 || c.pages <= 0 || c.pages > kMaxCount >> shift)
        return BNN_EINVAL;
    if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v))
        return BNN_EINVAL;
    const int64_t strides[6] = {c.k_page_stride, c.k_head_stride, c.k_row_stride,
                                c.v_page_stride, c.v_head_stride, c.v_row_stride};
    for (int64_t s : strides)
        if (s < c.head_dim || s % 8 != 0 || s >= ((int64_t)1 << 38))
            return BNN_EINVAL;
    *out = Cache{static_cast<unsigned char*>(c.k), static_cast<unsigned char*>(c.v), c.k_page_stride, c.k_head_stride,
                 c.k_row_stride, c.v_page_stride, c.v_head_stride, c.v_row_stride, (uint32_t)c.pages,
                 (uint32_t)c.kv_heads, shift};
    return BNN_OK;
}

// A launch that may start while the stream's previous kernel drains; every
// kernel here waits for it (griddep_wait) before it reads or writes memory.
template <typename Args>
BNN_Status launch(void (*kernel)(Args), dim3 grid, uint32_t threads, size_t smem, cudaStream_t stream, const Args& args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) {
        cudaGetLastError();
        return BNN_EIO;
    }
    return BNN_OK;
}

// The kernels here let their successor start early, and a one-row BNN job may
// read its input before it waits for its predecessor (GemvArgs::early_input):
// on the handle's own stream it must not while a paged call's outputs are in
// flight, that is until bnn_b200_sync or bnn_b200_paged_sync has drained it.
void outputs_in_flight(BNN_Device device, cudaStream_t stream) {
    if (stream == device->stream)
        device->inflight_overflow = true;
}

// ---- append

// (token, head) rows: more than the warps that fit the GPU's 148 SMs at once. One
// head a warp and four, 32 heads from FP32: 32 tokens 1.7 and 1.9 us, 64 2.0 and
// 1.9, 256 (8192 rows) 3.3 and 2.9, 512 4.8 and 3.4, 8192 69 and 32 (in a graph):
// the rule holds on to one head longer than it pays, by 0.5 us at most.
constexpr uint64_t kAppendWide = 148 * 64;

template <int D, typename S, typename T, int kHeads>
BNN_Status launch_append(const AppendArgs& a, bool interleaved, cudaStream_t stream) {
    constexpr uint32_t part = kHeads * (128 / D);
    const uint32_t parts = (a.heads + part - 1) / part + 2 * ((a.c.kv_heads + part - 1) / part);
    if (parts > 65535)
        return BNN_ENOTSUP;
    return launch(interleaved ? append_kernel<D, S, T, true, kHeads> : append_kernel<D, S, T, false, kHeads>,
                  dim3((a.tokens + kAppendThreads / 32 - 1) / (kAppendThreads / 32), parts), kAppendThreads, 0, stream, a);
}

template <int D, typename S, typename T>
BNN_Status append_heads(const AppendArgs& a, bool interleaved, cudaStream_t stream) {
    // Four heads a warp where that still fills the GPU (their loads overlap and
    // share the rotation's factors; two and eight were slower: 64 and 55 us against
    // 54 for 8192 tokens of 32 heads at the time), one where the call is short and
    // more warps are the faster way through it.
    const uint64_t rows = (uint64_t)a.tokens * (a.heads + 2 * a.c.kv_heads);
    return rows >= kAppendWide ? launch_append<D, S, T, 4>(a, interleaved, stream) : launch_append<D, S, T, 1>(a, interleaved, stream);
}

template <int D, typename T>
BNN_Status append_source(const AppendArgs& a, int64_t type, bool interleaved, cudaStream_t stream) {
    switch (type) {
    case BNN_PAGED_F32:
        return append_heads<D, float, T>(a, interleaved, stream);
    case BNN_PAGED_BF16:
        return append_heads<D, __nv_bfloat16, T>(a, interleaved, stream);
    default:
        return append_heads<D, __half, T>(a, interleaved, stream);
    }
}

// ---- attention

// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and
// device. BNN_DeviceOpen forgets what was allowed (bnn_paged_forget).
constexpr int kMaxDevices = 64, kMaxKernels = 16;
std::mutex g_allowed_mutex;
struct Allowed {
    const void* kernel;
    size_t bytes;
} g_allowed[kMaxDevices][kMaxKernels];

BNN_Status allow_smem(int ordinal, const void* kernel, size_t bytes) {
    if (ordinal < 0 || ordinal >= kMaxDevices)
        return BNN_ENOTSUP;
    std::lock_guard<std::mutex> lock(g_allowed_mutex);
    for (Allowed& e : g_allowed[ordinal]) {
        if (e.kernel != nullptr && e.kernel != kernel)
            continue;
        if (e.kernel == kernel && e.bytes >= bytes)
            return BNN_OK;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
            cudaGetLastError();
            return BNN_EIO;
        }
        e = Allowed{kernel, bytes};
        return BNN_OK;
    }
    return BNN_ENOTSUP;
}

// The workspace: for each CTA of the split kernel two records of partial rows,
// two of joined groups and four counters, zero between calls.
uint32_t split_grid(BNN_Device device) { return (uint32_t)device->sm_count * kDecPerSm; }
size_t partial_bytes(BNN_Device device) { return (size_t)split_grid(device) * 4 * DecodeShape<128>::kRecord * sizeof(float); }

size_t workspace_bytes(BNN_Device device) { return partial_bytes(device) + (size_t)split_grid(device) * 4 * sizeof(int); }

template <int D, typename T>
BNN_Status launch_split(BNN_Device device, const AttnArgs& a, cudaStream_t stream) {
    const size_t smem = decode_smem(DecodeShape<D>::kRingBytes, a.batch);
    const BNN_Status st = allow_smem(device->ordinal, (const void*)attention_split_kernel<D, T>, smem);
    if (st != BNN_OK)
        return st;
    // no more CTAs than blocks there can be
    const uint64_t per_row = (((uint64_t)a.table_width << a.c.page_shift) + kDecBlock - 1) / kDecBlock + 1;
    const uint64_t groups = ((uint64_t)a.max_q * a.group + kDecRows - 1) / kDecRows;
    const uint64_t most = (uint64_t)a.batch * a.c.kv_heads * (a.split_all ? groups : std::min(groups, (uint64_t)a.split_rows / kDecRows)) *
                          (per_row + kRowCost);
    if (most > INT32_MAX)
        return BNN_ENOTSUP;  // the shares' units are counted in 32 bits
    return launch(attention_split_kernel<D, T>, dim3((uint32_t)std::min<uint64_t>(split_grid(device), most)), kDecThreads, smem,
                  stream, a);
}

// The tensor map of one pool: columns, rows of a page, heads, pages; a box is
// 64 columns (the swizzle's 128 bytes) of up to 128 rows of one head's page.
BNN_Status encode_map(CUtensorMap* map, const void* base, bool half, uint32_t d, const Cache& c, int64_t page, int64_t head,
                      int64_t row) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<Encode>(fn);
    }();
    if (!encode)
        return BNN_ENOTSUP;
    const cuuint32_t rows = 1u << c.page_shift;
    const cuuint64_t dims[4] = {d, rows, c.kv_heads, c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[4] = {64, std::min<cuuint32_t>(rows, kPfKeys), 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult e = encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? BNN_OK : BNN_EIO;
}

template <int D, typename T, int kMode>
BNN_Status launch_tiles(BNN_Device device, const AttnArgs& a, cudaStream_t stream, bool every_request) {
    using Shape = PrefillShape<D, kMode>;
    constexpr bool half = std::is_same<T, __half>::value;
    PrefillArgs args;
    args.a = a;
    args.every_request = every_request;
    BNN_Status st = encode_map(&args.k_map, a.c.k, half, D, a.c, a.c.k_page, a.c.k_head, a.c.k_row);
    if (st == BNN_OK)
        st = encode_map(&args.v_map, a.c.v, half, D, a.c, a.c.v_page, a.c.v_head, a.c.v_row);
    if (st == BNN_OK)
        st = allow_smem(device->ordinal, (const void*)attention_tiles_kernel<D, T, kMode>, Shape::kSmem);
    if (st != BNN_OK)
        return st;
    const uint64_t items = ((uint64_t)a.tokens * a.group) / (Shape::kQTiles * kPfRows) + a.batch;  // at most
    if (items * a.c.kv_heads > INT32_MAX)
        return BNN_EINVAL;
    return launch(attention_tiles_kernel<D, T, kMode>, dim3((uint32_t)(items * a.c.kv_heads)), Shape::kThreads, Shape::kSmem,
                  stream, args);
}

// Positions from which requests of few rows get the split kernel beside tiles for
// the others. Tiles alone and both, in a graph: 60 single tokens behind 400 and a
// prompt of 512 66 and 46 us, behind 1000 97 and 67, behind 4000 277 and 179; but
// 8 single tokens and 100 tokens behind 400 12 and 25 us, behind 1000 19 and 31,
// behind 4000 56 and 81, where one kernel waits for the other and neither fills
// the GPU. How many requests there are of a kind only the device knows.
constexpr uint32_t kMixedCache = 1024;
// Positions up to which one stream works a tile of rows, in place of two in turn:
// prompts of 256 9.1 and 10.6 us, 512 12.3 and 12.9, 640 13.8 both, 768 15.5 and
// 15.0, 1024 18.6 and 17.1; 100 tokens behind 512 12.2 and 12.8, behind 768 15.3
// and 14.6.
constexpr uint32_t kTurnsCache = 512;

template <int D, typename T>
BNN_Status attention_typed(BNN_Device device, AttnArgs a, cudaStream_t stream) {
    // Requests of few rows go to the split kernel, the others to the tiles; each
    // kernel finds its own. The lengths are on the device: what a cache can be
    // long is the page table's width here, so a table that is wider than its
    // requests need can bring the other kernel, or both. Where one of them can serve the whole call it goes
    // alone (a launch that finds nothing to do costs 2 us): the split kernel if
    // no request has more than 16 rows, the tiles if every cache is short (eight
    // key tiles at most), either one for a single request.
    const uint64_t most_rows = (uint64_t)a.max_q * a.group;
    const bool long_cache = ((uint64_t)a.table_width << a.c.page_shift) >= kLongCache;
    a.split_rows = kDecRows * std::max<uint32_t>(1, kSplitGroups / (a.c.kv_heads * std::min(a.batch, kSplitGroups)));
    a.split_all = most_rows <= kDecRows || (long_cache && a.batch == 1 && most_rows <= a.split_rows);
    if (a.split_all)
        return launch_split<D, T>(device, a, stream);
    const bool mixed = a.batch > 1 && ((uint64_t)a.table_width << a.c.page_shift) >= kMixedCache;
    if (mixed) {
        const BNN_Status st = launch_split<D, T>(device, a, stream);
        if (st != BNN_OK)
            return st;
    }
    const uint64_t pairs = (((uint64_t)a.tokens * a.group) / (2 * kPfRows) + a.batch) * a.c.kv_heads;
    // Two row tiles in a CTA while such pairs fill the GPU; else one, with two
    // streams over its keys where there are enough of them (kTurnsCache; 256 tokens
    // behind 8192 positions 118 us with one stream and 93 with two).
    if (pairs >= (uint64_t)device->sm_count)
        return launch_tiles<D, T, kPair>(device, a, stream, !mixed);
    return ((uint64_t)a.table_width << a.c.page_shift) > kTurnsCache ? launch_tiles<D, T, kTurns>(device, a, stream, !mixed)
                                                                     : launch_tiles<D, T, kSingle>(device, a, stream, !mixed);
}

}  // namespace

namespace bnn {
cudaError_t set_test_hooks_paged(unsigned long long limit_ns, int starve) {
    cudaError_t e = cudaMemcpyToSymbol(g_wait_ns_limit, &limit_ns, sizeof limit_ns);
    if (e == cudaSuccess)
        e = cudaMemcpyToSymbol(paged::g_paged_starve, &starve, sizeof starve);
    return e;
}
}  // namespace bnn

void bnn_paged_forget(int ordinal) {
    if (ordinal < 0 || ordinal >= kMaxDevices)
        return;
    std::lock_guard<std::mutex> lock(g_allowed_mutex);
    for (Allowed& e : g_allowed[ordinal])
        e = Allowed{};
}

extern "C" {

BNN_Status bnn_b200_paged_append(BNN_Device device, const BNN_PagedAppend* desc, void* stream) {
    if (!device || !desc)
        return BNN_EINVAL;
    const BNN_PagedAppend& d = *desc;
    AppendArgs a = {};
    BNN_Status st = check_cache(d.cache, &a.c);
    if (st != BNN_OK)
        return st;
    if (d.type != BNN_PAGED_F32 && d.type != BNN_PAGED_BF16 && d.type != BNN_PAGED_F16)
        return BNN_EINVAL;
    if (d.tokens < 0 || d.tokens > kMaxCount || d.heads <= 0 || d.heads > 65536)
        return BNN_EINVAL;
    if (d.rotary_dim < 0 || d.rotary_dim > d.cache.head_dim)
        return BNN_EINVAL;
    if (d.rotary_dim % 8 != 0)
        return BNN_ENOTSUP;
    if (d.rotary_dim != 0 && (!d.cos || !d.sin || !aligned16(d.cos) || !aligned16(d.sin) || d.table_rows <= 0 || d.table_rows > kMaxCount))
        return BNN_EINVAL;
    if (!(d.eps >= 0.0) || !std::isfinite((float)d.eps) || !aligned16(d.q_norm) || !aligned16(d.k_norm))
        return BNN_EINVAL;
    if (d.tokens == 0)
        return BNN_OK;
    if (!d.q || !d.k || !d.v || !d.positions || !d.slots || !d.q_out)
        return BNN_EINVAL;
    if ((reinterpret_cast<uintptr_t>(d.q_out) & 7u) != 0 || d.out_token_stride % 4 != 0 || d.out_head_stride % 4 != 0)
        return BNN_EINVAL;
    a.src[0] = static_cast<const unsigned char*>(d.q);
    a.src[1] = static_cast<const unsigned char*>(d.k);
    a.src[2] = static_cast<const unsigned char*>(d.v);
    a.token[0] = d.q_token_stride;
    a.token[1] = d.k_token_stride;
    a.token[2] = d.v_token_stride;
    a.head[0] = d.q_head_stride;
    a.head[1] = d.k_head_stride;
    a.head[2] = d.v_head_stride;
    a.gain[0] = d.q_norm;
    a.gain[1] = d.k_norm;
    a.cos = d.cos;
    a.sin = d.sin;
    a.positions = d.positions;
    a.slots = d.slots;
    a.q_out = static_cast<unsigned char*>(d.q_out);
    a.o_token = d.out_token_stride;
    a.o_head = d.out_head_stride;
    a.tokens = (uint32_t)d.tokens;
    a.heads = (uint32_t)d.heads;
    a.rotary = (uint32_t)d.rotary_dim;
    a.table_rows = (uint32_t)d.table_rows;
    a.eps = (float)d.eps;
    a.status = device->d_status + bnn::kPagedStatusWord;
    bnn::DeviceGuard guard(device->ordinal);
    if (!guard.ok())
        return BNN_EIO;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = d.cache.head_dim == 128, inter = d.interleaved != 0;
    outputs_in_flight(device, s);
    if (d.cache.type == BNN_PAGED_BF16)
        return wide ? append_source<128, __nv_bfloat16>(a, d.type, inter, s)
                    : append_source<64, __nv_bfloat16>(a, d.type, inter, s);
    return wide ? append_source<128, __half>(a, d.type, inter, s) : append_source<64, __half>(a, d.type, inter, s);
}

BNN_Status bnn_b200_paged_workspace(BNN_Device device, size_t* bytes) {
    if (!device || !bytes)
        return BNN_EINVAL;
    *bytes = workspace_bytes(device);
    return BNN_OK;
}

BNN_Status bnn_b200_paged_attention(BNN_Device device, const BNN_PagedAttention* desc, void* stream) {
    if (!device || !desc)
        return BNN_EINVAL;
    const BNN_PagedAttention& d = *desc;
    AttnArgs a = {};
    BNN_Status st = check_cache(d.cache, &a.c);
    if (st != BNN_OK)
        return st;
    if (d.out_type != d.cache.type && d.out_type != BNN_PAGED_F32)
        return BNN_EINVAL;
    if (d.batch < 0 || d.tokens < 0 || d.tokens > kMaxCount || d.heads <= 0 || d.max_q < 0 || d.max_q > kMaxCount)
        return BNN_EINVAL;
    if (d.batch > BNN_PAGED_MAX_BATCH)
        return BNN_ENOTSUP;
    if (d.heads % d.cache.kv_heads != 0)
        return BNN_EINVAL;
    if (d.heads / d.cache.kv_heads > BNN_PAGED_MAX_GROUP)
        return BNN_ENOTSUP;
    const float scale_log2 = (float)(d.scale * 1.4426950408889634);
    if (d.window < 0 || d.sinks < 0 || !(d.scale > 0.0) || !std::isfinite(scale_log2) || (float)d.scale == 0.0f)
        return BNN_EINVAL;
    if (d.table_width < 0 || d.table_width > kMaxCount || (d.batch > 1 && d.table_stride < 0))
        return BNN_EINVAL;
    if (d.batch == 0 || d.tokens == 0 || d.max_q == 0)
        return BNN_OK;
    if (!d.q || !d.out || (!d.page_table && d.table_width) || !d.kv_lens || !d.q_starts || !d.workspace)
        return BNN_EINVAL;
    if (d.workspace_bytes < 0 || (size_t)d.workspace_bytes < workspace_bytes(device) || !aligned16(d.workspace))
        return BNN_EINVAL;
    a.q = static_cast<const unsigned char*>(d.q);
    a.out = static_cast<unsigned char*>(d.out);
    a.lse = d.lse;
    a.table = d.page_table;
    a.kv_lens = d.kv_lens;
    a.q_starts = d.q_starts;
    a.q_token = d.q_token_stride;
    a.q_head = d.q_head_stride;
    a.o_token = d.out_token_stride;
    a.o_head = d.out_head_stride;
    a.lse_token = d.lse_token_stride;
    a.table_stride = d.table_stride;
    a.batch = (uint32_t)d.batch;
    a.tokens = (uint32_t)d.tokens;
    a.heads = (uint32_t)d.heads;
    a.group = (uint32_t)(d.heads / d.cache.kv_heads);
    a.table_width = (uint32_t)d.table_width;
    a.max_q = (uint32_t)d.max_q;
    a.window = (uint32_t)(d.window < kMaxCount ? d.window : 0);  // a window past every position is none
    a.sinks = (uint32_t)(d.sinks < kMaxCount ? d.sinks : kMaxCount);
    a.out_type = (uint32_t)d.out_type;
    a.scale = (float)d.scale;
    a.scale_log2 = scale_log2;
    a.partials = static_cast<float*>(d.workspace);
    a.group_counters = reinterpret_cast<int*>(static_cast<unsigned char*>(d.workspace) + partial_bytes(device));
    a.row_counters = a.group_counters + 2 * split_grid(device);
    a.status = device->d_status + bnn::kPagedStatusWord;
    bnn::DeviceGuard guard(device->ordinal);
    if (!guard.ok())
        return BNN_EIO;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = d.cache.head_dim == 128;
    outputs_in_flight(device, s);
    if (d.cache.type == BNN_PAGED_BF16)
        return wide ? attention_typed<128, __nv_bfloat16>(device, a, s) : attention_typed<64, __nv_bfloat16>(device, a, s);
    return wide ? attention_typed<128, __half>(device, a, s) : attention_typed<64, __half>(device, a, s);
}

BNN_Status bnn_b200_paged_sync(BNN_Device device, void* stream) {
    if (!device)
        return BNN_EINVAL;
    bnn::DeviceGuard guard(device->ordinal);
    if (!guard.ok())
        return BNN_EIO;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int word = 0;
    if (cudaMemcpyAsync(&word, device->d_status + bnn::kPagedStatusWord, sizeof(int), cudaMemcpyDeviceToHost, s) !=
            cudaSuccess ||
        cudaMemsetAsync(device->d_status + bnn::kPagedStatusWord, 0, sizeof(int), s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess) {
        cudaGetLastError();
        return BNN_EIO;
    }
    if (s == device->stream)
        bnn::inflight_clear(device);
    if (word & bnn::kStatusTimeout)
        return BNN_ETIMEOUT;
    return word ? BNN_ERANGE : BNN_OK;
}

}  // extern "C"
