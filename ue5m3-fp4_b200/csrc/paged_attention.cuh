// Shared by the kernels of attention over a paged key/value cache: arguments, the row space, and
// how a sequence's keys are split over CTAs.
//
// Sequence b has query_starts[b + 1] - query_starts[b] = n new tokens; its cache holds
// kv_lengths[b] = L keys, the new ones included.  New token i stands at position L - n + i and sees
// the keys up to it; with L < n the first ones see none and their output is zero.  The G = heads /
// kv_heads query heads of one key/value head are rows of one matrix: row i * G + g is token i, head
// h * G + g, so that a tile of keys is read once for all of them.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "abi_common.cuh"
#include "tcgen05_ptx.cuh"

namespace ue5m3 {
namespace paged {

constexpr int kKeys = 64;  // keys per tile of the split, and of the small-rows kernel

struct Params {
    const __nv_bfloat16* q;
    int64_t q_token, q_head;     // strides in elements
    __nv_bfloat16* out;          // [tokens, heads, head_dim]
    const int* page_table;       // [sequences, table_width]
    int64_t table_stride;
    const int* kv_lengths;
    const int* query_starts;
    const __nv_bfloat16* v_pages;
    int64_t v_page, v_slot, v_head;
    float* partial;              // [tokens, heads, splits, head_dim], then [tokens, heads, splits, 2]
    int* status;
    int sequences, tokens, heads, kv_heads, group;
    int table_width, pages, page_shift;
    int chunk;                   // key tiles per split
    int splits;                  // splits that the grid and the workspace have room for
    int zero_tail;               // rows behind the last sequence are set to zero
    float scale_log2;            // scale * log2(e)
};

struct Sequence {
    int first;   // row of q of its first new token
    int queries; // new tokens
    int keys;    // keys in the cache, no more than the page table has room for
    bool cut;    // kv_lengths says more than the table has room for
};

__device__ __forceinline__ Sequence sequence_of(const Params& p, int b) {
    Sequence s;
    const int start = min(max(p.query_starts[b], 0), p.tokens);
    const int stop = min(max(p.query_starts[b + 1], start), p.tokens);
    s.first = start;
    s.queries = stop - start;
    const int64_t room = (int64_t)p.table_width << p.page_shift;
    const int length = max(p.kv_lengths[b], 0);
    s.cut = length > room;
    s.keys = s.cut ? (int)room : length;
    return s;
}

// keys that the last of rows row0 ... row0 + count - 1 sees (the most that any of them sees)
__device__ __forceinline__ int visible_keys(const Params& p, const Sequence& s, int row0, int count) {
    const int last = min(s.queries - 1, (row0 + count - 1) / p.group);
    return max(0, s.keys - s.queries + last + 1);
}

// key tiles per split for a row tile that sees `tiles` of them, an even number if the plan's is
__device__ __forceinline__ int split_chunk(const Params& p, int tiles) {
    const int least = (tiles + p.splits - 1) / p.splits;
    return max(p.chunk, p.chunk & 1 ? least : (least + 1) & ~1);
}

// The page of a key, or -1 where the table names none of the cache's.
__device__ __forceinline__ int page_of(const Params& p, int b, int key) {
    const int page = __ldg(p.page_table + (int64_t)b * p.table_stride + (key >> p.page_shift));
    return page >= 0 && page < p.pages ? page : -1;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y,
                                            int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(ptx::smem_u32(dst)), "l"(map), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// rows of q behind the last sequence
__device__ __forceinline__ void zero_tail_rows(const Params& p, int64_t thread, int64_t threads, int head_dim) {
    const int64_t width = (int64_t)p.heads * head_dim / 8;  // 16-byte pieces of a row
    const int first = min(max(p.query_starts[p.sequences], 0), p.tokens);
    uint4* out = reinterpret_cast<uint4*>(p.out);
    for (int64_t i = first * width + thread; i < p.tokens * width; i += threads) out[i] = make_uint4(0, 0, 0, 0);
}

// Values that not every row of a tile sees may be infinite or NaN: a product with the others' zeros
// would spread them.  Whether one of two bf16 in a word is not finite:
__device__ __forceinline__ bool odd_pair(uint32_t w) {
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}
__device__ __forceinline__ bool odd_piece(const uint4& v) {
    return odd_pair(v.x) || odd_pair(v.y) || odd_pair(v.z) || odd_pair(v.w);
}

template <typename... Arguments>
cudaError_t launch_after(void (*kernel)(Arguments...), dim3 grid, unsigned threads, size_t shared, cudaStream_t stream,
                         bool early, Arguments... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, arguments...);
}

// mbar_wait with one answer for the whole (converged) warp
__device__ __forceinline__ bool warp_wait(unsigned long long* bar, uint32_t parity, int* abort_flag, int* status, int where,
                                          int iter) {
    return __all_sync(0xFFFFFFFFu, ptx::mbar_wait(bar, parity, abort_flag, status, where, iter));
}

// ---- the kernel for many rows (paged_attention_wide.cu) ------------------------------------------

constexpr int kWideRows = 256;  // rows of one CTA

// early: the kernel launched before it on the stream belongs to the same call
int launch_wide(const Params& p, int head_dim, dim3 grid, const CUtensorMap& k_map, const CUtensorMap& v_map, bool early,
                cudaStream_t stream);

}  // namespace paged
}  // namespace ue5m3
