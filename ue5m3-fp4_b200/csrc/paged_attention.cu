// Attention of a chunk of new tokens over a paged key/value cache: the kernel for few rows per
// key/value head (single tokens above all), the write of the new keys and values into their
// pages, and the C entry point.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
//
// One pass over the keys with the running maximum and sum of the softmax; both and the output row
// are held in fp32, the probabilities are rounded to bf16 for their product with v (the products'
// own type; the sum takes them unrounded).
//
// What bounds it: reading K and V once (4 * head_dim bytes per key and key/value head).  One CTA
// owns up to 16 rows (the query heads of a key/value head) and a run of keys; TMA brings 64 keys of
// K and V per stage, page by page, into three 128-byte-swizzled stages; four warps take 16 keys of
// a stage each, with a running maximum, sum and output of their own (mma.m16n8k16), which meet in
// shared memory at the end of the run.  Long sequences are split over CTAs, which leave their
// unnormalised rows in a workspace for a second, short launch.
//
// Measured, 32 heads over 4 key/value heads of 128: 64 tokens of up to 8192 keys each, 522 MB: 103 us,
// 5.1 TB/s of 6.5; one token of 32768 keys, 67 MB: 24.7 us, 2.7 TB/s, of which about 10 us are the two
// launches, the first page's address and data, the merge and the combination of the splits.
#include <cudaTypedefs.h>
#include <math.h>

#include "abi_common.cuh"
#include "paged_attention.cuh"
#include "tcgen05_ptx.cuh"

namespace ue5m3 {
namespace paged {

constexpr int kRows = 16;
constexpr int kStages = 3;
constexpr int kConsumers = 4;
constexpr int kSmallThreads = (kConsumers + 1) * 32;
constexpr int kSiteFull = 0x50, kSiteEmpty = 0x51;

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- new keys and values into their pages -------------------------------------------------------

struct AppendParams {
    const __nv_bfloat16 *k, *v;
    int64_t k_token, k_head, v_token, v_head;
    __nv_bfloat16 *k_pages, *v_pages;
    int64_t k_page, k_slot, k_page_head, v_page, v_slot, v_page_head;
};

// One 16-byte piece of a new token's key and value.  Token `token` of the sequence, whose place is
// key `position`; a page that is not one of the cache's is left out.
__device__ __forceinline__ void append_piece(const Params& p, const AppendParams& a, const Sequence& s, int b, int token,
                                             int position, int head, int piece) {
    const int page = page_of(p, b, position);
    if (page < 0) return;
    const int slot = position & ((1 << p.page_shift) - 1);
    const int64_t row = s.first + token;
    const uint4 k = *reinterpret_cast<const uint4*>(a.k + row * a.k_token + head * a.k_head + piece * 8);
    const uint4 v = *reinterpret_cast<const uint4*>(a.v + row * a.v_token + head * a.v_head + piece * 8);
    *reinterpret_cast<uint4*>(a.k_pages + page * a.k_page + slot * a.k_slot + head * a.k_page_head + piece * 8) = k;
    *reinterpret_cast<uint4*>(a.v_pages + page * a.v_page + slot * a.v_slot + head * a.v_page_head + piece * 8) = v;
}

// Before the kernel for many rows, whose CTAs read one another's new keys: one thread per piece, the
// threads of a block run over (token, head, piece) of one sequence.  Bound by memory, 8 * head_dim
// bytes per token and head; 2048 tokens of 4 heads are 8 MB, about 2 us next to the 235 that follow.
template <int kDim>
__global__ void __launch_bounds__(256) append_kernel(const Params p, const AppendParams a) {
    constexpr int kPieces = kDim / 8;
    launch_dependents();
    const int b = blockIdx.y;
    const Sequence s = sequence_of(p, b);
    if (s.cut) return;  // no place in the table
    const int64_t count = (int64_t)s.queries * p.kv_heads * kPieces;
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) {
        const int piece = (int)(i % kPieces), head = (int)(i / kPieces % p.kv_heads), token = (int)(i / kPieces / p.kv_heads);
        const int position = s.keys - s.queries + token;
        if (position >= 0) append_piece(p, a, s, b, token, position, head, piece);
    }
}

// ---- few rows -------------------------------------------------------------------------------------

template <int kDim>
struct SmallShared {
    static constexpr int kTileBytes = kKeys * kDim * 2;  // K or V of a stage: kDim / 64 slabs of [64 keys][128 bytes]
    static constexpr int kBytes = kStages * 2 * kTileBytes + 1024 + 256;
};

template <int kDim>
__global__ void __launch_bounds__(kSmallThreads, 2)
    attention_small_kernel(const Params p, const AppendParams append, const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map) {
    constexpr int kSlabs = kDim / 64, kSteps = kDim / 16;
    constexpr int kTileBytes = SmallShared<kDim>::kTileBytes;
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned long long* full = reinterpret_cast<unsigned long long*>(tiles + kStages * 2 * kTileBytes);
    unsigned long long* empty = full + kStages;
    int* abort_flag = reinterpret_cast<int*>(empty + kStages);
    int* bad = abort_flag + 1;
    constexpr int kMergeRow = kDim + 4;  // a row's channels, its maximum and sum, on a 16-byte boundary
    float* merge = reinterpret_cast<float*>(tiles);  // after the last stage: [warp][16 rows][kMergeRow]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z;
    const int row_tiles = gridDim.y / p.kv_heads;
    const int head = blockIdx.y / row_tiles;
    const Sequence s = sequence_of(p, b);
    const int rows = s.queries * p.group;
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], kConsumers);
        }
        *abort_flag = p.status && *((volatile int*)p.status) != 0;  // a recorded failure: no work, NaN
        ptx::mbar_fence_init();
    }
    __syncthreads();
    int issue = 0;  // stages filled (producer) or read (consumers) so far
    for (int row0 = (blockIdx.y % row_tiles) * kRows; row0 < rows; row0 += row_tiles * kRows) {
        const int limit = visible_keys(p, s, row0, kRows);
        const int all = (limit + kKeys - 1) / kKeys;
        const int chunk = split_chunk(p, all);
        const int first = blockIdx.x * chunk, last = min(all, first + chunk);
        const int splits = (all + chunk - 1) / chunk;
        if (first >= all && blockIdx.x > 0) continue;
        if (append.k && !s.cut) {
            // The new tokens among this CTA's keys go to their pages; it alone reads them before the
            // call ends, or, with a second row tile, next to one that writes the same.
            constexpr int kPieces = kDim / 8;
            const int start = max(s.keys - s.queries, first * kKeys), stop = min(limit, (first + chunk) * kKeys);
            for (int i = threadIdx.x; i < (stop - start) * kPieces; i += kSmallThreads)
                append_piece(p, append, s, b, start + i / kPieces - (s.keys - s.queries), start + i / kPieces, head, i % kPieces);
            asm volatile("fence.proxy.async;" ::: "memory");
        }
        if (threadIdx.x == 0) *bad = s.cut;
        __syncthreads();
        const bool dead = *((volatile int*)abort_flag) != 0;  // a wait gave up, here or in an earlier launch
        if (dead) {
        } else if (warp == kConsumers) {
            // TMA: lane i brings the i-th page's share of the tile
            const int box = min(kKeys, 1 << p.page_shift), boxes = kKeys / box;
            for (int tile = first; tile < last; ++tile, ++issue) {
                const int stage = issue % kStages;
                if (issue >= kStages && !warp_wait(&empty[stage], ((issue / kStages) & 1) ^ 1, abort_flag,
                                                        p.status, kSiteEmpty, issue))
                    break;
                const int key = tile * kKeys + lane * box;
                const bool wanted = lane < boxes && key < limit;
                const int page = wanted ? page_of(p, b, key) : -1;
                if (wanted && page < 0) *bad = 1;
                const uint32_t loads = __ballot_sync(0xFFFFFFFFu, page >= 0);
                if (lane == 0)
                    ptx::mbar_arrive_expect_tx(&full[stage], __popc(loads) * box * kDim * 2 * 2);
                __syncwarp();
                if (page >= 0) {
                    unsigned char* k = tiles + stage * 2 * kTileBytes + lane * box * 128;
                    unsigned char* v = k + kTileBytes;
                    const int slot = key & ((1 << p.page_shift) - 1);
#pragma unroll
                    for (int i = 0; i < kSlabs; ++i) {
                        tma_load_4d(k + i * kKeys * 128, &k_map, &full[stage], i * 64, head, slot, page);
                        tma_load_4d(v + i * kKeys * 128, &v_map, &full[stage], i * 64, head, slot, page);
                    }
                }
            }
            if (*((volatile int*)abort_flag))  // copies in flight land before their memory is used otherwise
                for (int i = max(0, issue - kStages); i < issue; ++i)
                    for (int spin = 0; spin < 1000000 && !ptx::mbar_try_wait(&full[i % kStages], (i / kStages) & 1);)
                        ++spin;
        } else {
            const int g = lane >> 2, c = lane & 3;
            uint32_t q[kSteps][4];
            int last_key[2];  // the last key that rows g and g + 8 see
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = row0 + g + 8 * h;
                const int token = r / p.group;
                last_key[h] = r < rows ? s.keys - s.queries + token : -1;
                const __nv_bfloat16* source =
                    p.q + (int64_t)(s.first + token) * p.q_token + (int64_t)(head * p.group + r % p.group) * p.q_head;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    q[i][h] = r < rows ? *reinterpret_cast<const uint32_t*>(source + i * 16 + 2 * c) : 0;
                    q[i][h + 2] = r < rows ? *reinterpret_cast<const uint32_t*>(source + i * 16 + 8 + 2 * c) : 0;
                }
            }
            float o[kDim / 8][4];
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
            const int fewest = visible_keys(p, s, row0, 1);  // keys that every row sees
            for (int tile = first; tile < last; ++tile, ++issue) {
                const int stage = issue % kStages;
                if (!warp_wait(&full[stage], (issue / kStages) & 1, abort_flag, p.status, kSiteFull, issue)) break;
                unsigned char* k = tiles + stage * 2 * kTileBytes;
                unsigned char* v = k + kTileBytes;
                const int key0 = tile * kKeys + warp * 16;  // this warp's keys
                if (key0 + 16 > limit) {
                    // rows of V that no row sees may hold anything: 0 * NaN is not 0
                    for (int i = lane; i < 16 * kSlabs * 8; i += 32) {
                        const int key = i / (kSlabs * 8), piece = i % (kSlabs * 8);
                        if (key0 + key >= limit)
                            *reinterpret_cast<uint4*>(v + (piece / 8) * kKeys * 128 + (warp * 16 + key) * 128 +
                                                      (((piece & 7) ^ (key & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async;" ::: "memory");  // TMA may write this stage again
                    __syncwarp();
                }
                float score[2][4] = {};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    uint32_t kb[4];
                    const int key = warp * 16 + (lane >> 4) * 8 + (lane & 7), piece = i * 2 + ((lane >> 3) & 1);
                    ldmatrix_x4(kb, ptx::smem_u32(k) + (piece / 8) * kKeys * 128 + key * 128 +
                                        (((piece & 7) ^ (key & 7)) << 4));
                    mma_bf16(score[0], q[i], kb[0], kb[1]);
                    mma_bf16(score[1], q[i], kb[2], kb[3]);
                }
                uint32_t pr[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float now = -INFINITY;
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + (i >> 1) * 8 + 2 * c + (i & 1);
                        x[i] = key <= last_key[h] ? score[i >> 1][2 * h + (i & 1)] * p.scale_log2 : -INFINITY;
                        now = fmaxf(now, x[i]);
                    }
                    now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, 1));
                    now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, 2));
                    now = fmaxf(now, top[h]);
                    const float base = now == -INFINITY ? 0.0f : now;
                    const float fade = exp2_approx(top[h] - base);
                    float add = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = exp2_approx(x[i] - base);
                        add += x[i];
                    }
                    pr[h] = pack_bf16(x[0], x[1]);
                    pr[h + 2] = pack_bf16(x[2], x[3]);
                    sum[h] = __fmaf_rn(sum[h], fade, add);
                    top[h] = now;
#pragma unroll
                    for (int i = 0; i < kDim / 8; ++i) {
                        o[i][2 * h] *= fade;
                        o[i][2 * h + 1] *= fade;
                    }
                }
                // keys that some rows do not see: are their values finite?
                bool odd = false;
                if (key0 + 16 > fewest && fewest < limit)
                    for (int i = lane; i < 16 * kSlabs * 8; i += 32) {
                        const int key = i / (kSlabs * 8), piece = i % (kSlabs * 8);
                        odd |= key0 + key >= fewest &&
                               odd_piece(*reinterpret_cast<const uint4*>(v + (piece / 8) * kKeys * 128 + (warp * 16 + key) * 128 +
                                                                         ((piece & 7) << 4)));
                    }
                if (__any_sync(0xFFFFFFFFu, odd)) {
                    // seldom: one key after the other, for the rows that see it
                    for (int key = 0; key < 16; ++key) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t pair = __shfl_sync(0xFFFFFFFFu, pr[h + (key & 8 ? 2 : 0)], (lane & 28) + (key & 7) / 2);
                            const float weight = __uint_as_float(key & 1 ? pair & 0xFFFF0000u : pair << 16);
                            if (key0 + key > last_key[h]) continue;
#pragma unroll
                            for (int i = 0; i < kDim / 8; ++i) {
                                const uint32_t word = *reinterpret_cast<const uint32_t*>(
                                    v + (i / 8) * kKeys * 128 + (warp * 16 + key) * 128 + (((i & 7) ^ (key & 7)) << 4) + 4 * c);
                                o[i][2 * h] = __fmaf_rn(weight, __uint_as_float(word << 16), o[i][2 * h]);
                                o[i][2 * h + 1] = __fmaf_rn(weight, __uint_as_float(word & 0xFFFF0000u), o[i][2 * h + 1]);
                            }
                        }
                        __syncwarp();
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kDim / 16; ++i) {
                        uint32_t vb[4];
                        const int key = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), piece = i * 2 + (lane >> 4);
                        ldmatrix_x4_trans(vb, ptx::smem_u32(v) + (piece / 8) * kKeys * 128 + key * 128 +
                                                  (((piece & 7) ^ (key & 7)) << 4));
                        mma_bf16(o[2 * i], pr, vb[0], vb[1]);
                        mma_bf16(o[2 * i + 1], pr, vb[2], vb[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&empty[stage]);
            }
            // all warps' stages are read: the tiles' memory takes the four partial rows
            asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 2);
                float* to = merge + (warp * kRows + g + 8 * h) * kMergeRow;
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i)
                    *reinterpret_cast<float2*>(to + i * 8 + 2 * c) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
                if (c == 0) {
                    to[kDim] = top[h];
                    to[kDim + 1] = sum[h];
                }
            }
        }
        __syncthreads();
        const bool failed = *((volatile int*)abort_flag) || *((volatile int*)bad);
        for (int i = threadIdx.x; i < kRows * (kDim / 4); i += kSmallThreads) {
            const int r = i / (kDim / 4), d = i % (kDim / 4) * 4;
            if (row0 + r >= rows) continue;
            float most = -INFINITY, total = 0.0f;
            float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (failed) {
                most = 0.0f;
                value.x = value.y = value.z = value.w = total = __uint_as_float(0x7FC00000u);
            } else {
                const float* from = merge + r * kMergeRow;
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) most = fmaxf(most, from[w * kRows * kMergeRow + kDim]);
                const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(from + w * kRows * kMergeRow + d);
                    const float weight = exp2_approx(from[w * kRows * kMergeRow + kDim] - base);
                    total = __fmaf_rn(from[w * kRows * kMergeRow + kDim + 1], weight, total);
                    value.x = __fmaf_rn(v.x, weight, value.x);
                    value.y = __fmaf_rn(v.y, weight, value.y);
                    value.z = __fmaf_rn(v.z, weight, value.z);
                    value.w = __fmaf_rn(v.w, weight, value.w);
                }
            }
            const int token = (row0 + r) / p.group;
            const int64_t at = (int64_t)(s.first + token) * p.heads + head * p.group + (row0 + r - token * p.group);
            if (splits <= 1) {
                const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
                *reinterpret_cast<uint2*>(p.out + at * kDim + d) =
                    make_uint2(pack_bf16(value.x * inverse, value.y * inverse), pack_bf16(value.z * inverse, value.w * inverse));
            } else {
                const int64_t slot = at * p.splits + blockIdx.x;
                *reinterpret_cast<float4*>(p.partial + slot * kDim + d) = value;
                if (d == 0)
                    *reinterpret_cast<float2*>(p.partial + (int64_t)p.tokens * p.heads * p.splits * kDim + slot * 2) =
                        make_float2(most, total);
            }
        }
        // the merge memory is the next row tile's first stages
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncthreads();
    }
    if (p.zero_tail)
        zero_tail_rows(p, ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kSmallThreads + threadIdx.x,
                       (int64_t)gridDim.x * gridDim.y * gridDim.z * kSmallThreads, kDim);
}

// The rows of a split sequence: sum of the splits' rows, each faded to the largest maximum.  Few
// splits: one warp per (token, head), kDim / 32 channels per lane.
template <int kDim>
__global__ void __launch_bounds__(256) combine_few_kernel(const Params p, int rows_per_tile) {
    constexpr int kOwn = kDim / 32;
    wait_for_launcher();
    const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Sequence s = sequence_of(p, b);
    for (int i = blockIdx.x * 8 + warp; i < s.queries * p.heads; i += gridDim.x * 8) {
        const int token = i / p.heads, head = i - token * p.heads;
        const int row = token * p.group + head % p.group;
        const int all = (visible_keys(p, s, row / rows_per_tile * rows_per_tile, rows_per_tile) + kKeys - 1) / kKeys;
        const int chunk = split_chunk(p, all), splits = (all + chunk - 1) / max(chunk, 1);
        if (splits <= 1) continue;  // written by its only split
        const int64_t at = (int64_t)(s.first + token) * p.heads + head;
        const float* rows = p.partial + at * p.splits * kDim + lane * kOwn;
        const float2* stats =
            reinterpret_cast<const float2*>(p.partial + (int64_t)p.tokens * p.heads * p.splits * kDim + at * p.splits * 2);
        const float2 mine = lane < splits ? stats[lane] : make_float2(-INFINITY, 0.0f);
        float most = mine.x;
#pragma unroll
        for (int m = 16; m; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        const float weight = exp2_approx(mine.x - (most == -INFINITY ? 0.0f : most));
        float total = mine.y * weight;
#pragma unroll
        for (int m = 16; m; m >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, m);
        float value[kOwn] = {};
#pragma unroll 4
        for (int j = 0; j < splits; ++j) {
            const float w = __shfl_sync(0xFFFFFFFFu, weight, j);
            float v[kOwn];
            if constexpr (kOwn == 4)
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(rows + (int64_t)j * kDim);
            else
                *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(rows + (int64_t)j * kDim);
#pragma unroll
            for (int e = 0; e < kOwn; ++e) value[e] = __fmaf_rn(v[e], w, value[e]);
        }
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        uint32_t* out = reinterpret_cast<uint32_t*>(p.out + at * kDim + lane * kOwn);
#pragma unroll
        for (int e = 0; e < kOwn; e += 2) out[e / 2] = pack_bf16(value[e] * inverse, value[e + 1] * inverse);
    }
}

// Many splits: one CTA per (token, head), a quarter of the splits per warp, four channels per lane
// (head_dim 64: two splits side by side in a warp).
template <int kDim>
__global__ void __launch_bounds__(128) combine_kernel(const Params p, int rows_per_tile) {
    wait_for_launcher();
    constexpr int kLanes = kDim / 4, kSide = 128 / kLanes;  // lanes of a row, rows side by side in the CTA
    __shared__ float values[kSide][kDim], sums[kSide], tops[4];
    const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int side = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    const Sequence s = sequence_of(p, b);
    for (int i = blockIdx.x; i < s.queries * p.heads; i += gridDim.x) {
        const int token = i / p.heads, head = i % p.heads;
        const int row = token * p.group + head % p.group;
        const int all = (visible_keys(p, s, row / rows_per_tile * rows_per_tile, rows_per_tile) + kKeys - 1) / kKeys;
        const int chunk = split_chunk(p, all), splits = (all + chunk - 1) / max(chunk, 1);
        if (splits <= 1) continue;  // written by its only split
        const int64_t at = (int64_t)(s.first + token) * p.heads + head;
        const float* rows = p.partial + at * p.splits * kDim;
        const float* stats = p.partial + (int64_t)p.tokens * p.heads * p.splits * kDim + at * p.splits * 2;
        float most = -INFINITY;
        for (int j = threadIdx.x; j < splits; j += 128) most = fmaxf(most, stats[2 * j]);
#pragma unroll
        for (int m = 16; m; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        if (lane == 0) tops[warp] = most;
        __syncthreads();
        most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float base = most == -INFINITY ? 0.0f : most;
        float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float total = 0.0f;
#pragma unroll 4
        for (int j = side; j < splits; j += kSide) {
            const float4 v = *reinterpret_cast<const float4*>(rows + (int64_t)j * kDim + d);
            const float weight = exp2_approx(stats[2 * j] - base);
            total = __fmaf_rn(stats[2 * j + 1], weight, total);
            value.x = __fmaf_rn(v.x, weight, value.x);
            value.y = __fmaf_rn(v.y, weight, value.y);
            value.z = __fmaf_rn(v.z, weight, value.z);
            value.w = __fmaf_rn(v.w, weight, value.w);
        }
        *reinterpret_cast<float4*>(&values[side][d]) = value;
        if (d == 0) sums[side] = total;
        __syncthreads();
        if (threadIdx.x < kDim) {
            float v = 0.0f, t = 0.0f;
#pragma unroll
            for (int j = 0; j < kSide; ++j) {
                v += values[j][threadIdx.x];
                t += sums[j];
            }
            p.out[at * kDim + threadIdx.x] = __float2bfloat16_rn(t == 0.0f ? 0.0f : v / t);
        }
        __syncthreads();
    }
}

// ---- host -----------------------------------------------------------------------------------------

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        void* pointer = nullptr;
        cudaDriverEntryPointQueryResult query;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &query) != cudaSuccess ||
            query != cudaDriverEntryPointSuccess)
            return nullptr;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(pointer);
    }
    return fn;
}

// pages [page][slot][head][dim] as boxes of 64 channels of one head over `box` slots of one page
static int encode_pages(CUtensorMap* map, const void* base, const ue5m3_paged_cache& cache, int64_t page_stride,
                        int64_t slot_stride, int64_t head_stride, int head_dim, int box) {
    PFN_cuTensorMapEncodeTiled_v12000 encode = encode_fn();
    if (!encode) {
        record_error_text("cuTensorMapEncodeTiled is not available from the driver");
        return UE5M3_ERR_CUDA;
    }
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)cache.kv_heads, (cuuint64_t)cache.page_size,
                                (cuuint64_t)cache.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)head_stride * 2, (cuuint64_t)slot_stride * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    const CUresult result =
        encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, boxes, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS) {
        record_error_text("cuTensorMapEncodeTiled failed for the cache's pages");
        return UE5M3_ERR_CUDA;
    }
    return UE5M3_OK;
}

struct Plan {
    bool wide;
    int row_tiles;  // per sequence and key/value head, at most
    int chunk, splits;
    size_t workspace;
};

static size_t workspace_of(int64_t tokens, int64_t heads, int64_t head_dim, int64_t splits) {
    return splits > 1 ? (size_t)tokens * heads * splits * (head_dim + 2) * sizeof(float) : 0;
}

// Up to 32 rows per key/value head: the kernel for few rows, whose 16-row tiles read the keys once
// each (32 rows, 16 sequences of 4096 keys: 44 us against 70; one of 32768: 26 against 34); more: the
// tensor-core kernel with its 256-row tiles (64 rows, the same: 71 us against 76, 35 against 42).
// Splits of the keys: few rows, enough CTAs for two on every SM, runs of 4 to 16 tiles.  Many rows:
// one CTA per SM at most, runs of at least 8 tiles, and no more than pays: a split takes its share of about 0.93 us per 64 keys off the
// time and adds the writing and reading of its partial rows at about 0.7 TB/s, so that the square
// root of their quotient is the best number (8 x 32 heads over 32768 keys: 465 -> 35 us with 37 splits;
// 4 x 128 tokens over 2048 keys: 46.5 us without, 57.8 with 3).
// One plan serves the whole call and goes by its longest query and sequence: single tokens behind long
// contexts are split as finely as they need only in a call without a prompt chunk.
static Plan make_plan(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
                      int64_t max_query, int64_t max_kv) {
    Plan plan;
    const int64_t rows = max_query * (heads / kv_heads), sms = sm_count();
    plan.wide = rows > 2 * kRows;
    const int64_t tile_rows = plan.wide ? kWideRows : kRows;
    int64_t tiles = (rows + tile_rows - 1) / tile_rows;
    if (tiles * kv_heads > 65535) tiles = 65535 / kv_heads;
    plan.row_tiles = (int)tiles;
    const int64_t all = (max_kv + kKeys - 1) / kKeys, lists = sequences * kv_heads * tiles;
    int64_t chunk, splits;
    if (plan.wide) {
        const double whole = 0.93e-6 * (double)all, each = (double)(tokens * heads * (head_dim + 2) * 4) / 0.7e12;
        const int64_t most = (sms + lists - 1) / lists, best = (int64_t)sqrt(whole / each);
        const int64_t wanted = best < 1 || most < 2 ? 1 : best < most ? best : most;
        chunk = (all + wanted - 1) / wanted;
        chunk = ((chunk < 8 ? 8 : chunk) + 1) / 2 * 2;  // whole 128-key tiles
        splits = (all + chunk - 1) / chunk;
    } else {
        chunk = (all * lists + 2 * sms - 1) / (2 * sms);
        chunk = chunk < 4 ? 4 : chunk > 16 ? 16 : chunk;
        splits = (all + chunk - 1) / chunk;
    }
    plan.chunk = (int)chunk;
    plan.splits = (int)splits;
    plan.workspace = workspace_of(tokens, heads, head_dim, splits);
    return plan;
}

template <int kDim>
int launch(const Params& p, const Plan& plan, const CUtensorMap& k_map, const CUtensorMap& v_map, const AppendParams& append,
           int64_t max_query, cudaStream_t stream) {
    const dim3 grid(plan.splits, p.kv_heads * plan.row_tiles, p.sequences);
    cudaError_t error;
    if (plan.wide) {
        if (append.k) {
            const int64_t pieces = max_query * p.kv_heads * (kDim / 8);
            int64_t blocks = (pieces + 255) / 256;
            if (blocks > 1024) blocks = 1024;
            append_kernel<kDim><<<dim3((unsigned)blocks, p.sequences), 256, 0, stream>>>(p, append);
            const int status = check_launch();
            if (status != UE5M3_OK) return status;
        }
        const int status = launch_wide(p, kDim, grid, k_map, v_map, append.k != nullptr, stream);
        if (status != UE5M3_OK) return status;
    } else {
        error = allow_shared<attention_small_kernel<kDim>>(SmallShared<kDim>::kBytes);
        if (error == cudaSuccess)
            error = launch_after(attention_small_kernel<kDim>, grid, kSmallThreads, SmallShared<kDim>::kBytes, stream, false, p,
                                 append, k_map, v_map);
        if (error != cudaSuccess) return record_cuda_error(error);
    }
    if (plan.splits == 1) return UE5M3_OK;
    int64_t blocks = max_query * p.heads;
    const int tile_rows = plan.wide ? kWideRows : kRows;
    if (plan.splits <= 16) {
        blocks = (blocks + 7) / 8;
        if (blocks > 65535) blocks = 65535;
        error = launch_after(combine_few_kernel<kDim>, dim3((unsigned)blocks, p.sequences), 256, 0, stream, true, p, tile_rows);
    } else {
        if (blocks > 65535) blocks = 65535;
        error = launch_after(combine_kernel<kDim>, dim3((unsigned)blocks, p.sequences), 128, 0, stream, true, p, tile_rows);
    }
    return record_cuda_error(error);
}

}  // namespace paged
}  // namespace ue5m3

static bool paged_sizes_ok(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t head_dim,
                           int64_t max_query, int64_t max_kv) {
    return tokens > 0 && sequences > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 &&
           (head_dim == 64 || head_dim == 128) && max_query > 0 && max_kv > 0;
}

extern "C" size_t ue5m3_paged_attention_workspace_bytes(int64_t tokens, int64_t sequences, int64_t heads,
                                                        int64_t kv_heads, int64_t head_dim, int64_t max_query,
                                                        int64_t max_kv) {
    if (!paged_sizes_ok(tokens, sequences, heads, kv_heads, head_dim, max_query, max_kv)) return 0;
    return ue5m3::paged::make_plan(tokens, sequences, heads, kv_heads, head_dim, max_query, max_kv).workspace;
}

extern "C" int ue5m3_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                                     int64_t heads, const ue5m3_paged_cache* cache, const int* kv_lengths,
                                     const int* query_starts, int64_t max_query, int64_t max_kv, float scale,
                                     const void* new_k, int64_t new_k_token_stride, int64_t new_k_head_stride,
                                     const void* new_v, int64_t new_v_token_stride, int64_t new_v_head_stride, void* out,
                                     int zero_tail, void* workspace, size_t workspace_bytes, int* status_dev,
                                     void* stream) {
    using namespace ue5m3;
    using namespace ue5m3::paged;
    if (!q || !cache || !kv_lengths || !query_starts || !out || !cache->k_pages || !cache->v_pages ||
        !cache->page_table || (new_k == nullptr) != (new_v == nullptr) || !(scale > 0.0f) || scale > 0x1p126f)
        return UE5M3_ERR_INVALID_ARGUMENT;
    const int64_t dim = cache->head_dim;
    if (!paged_sizes_ok(tokens, cache->sequences, heads, cache->kv_heads, dim, max_query, max_kv) || cache->pages <= 0 ||
        cache->table_width <= 0 || cache->table_stride < cache->table_width)
        return UE5M3_ERR_INVALID_ARGUMENT;
    const int64_t page = cache->page_size;
    if (page < 16 || page > 256 || (page & (page - 1))) {
        record_error_text("page_size must be 16, 32, 64, 128 or 256");
        return UE5M3_ERR_UNSUPPORTED;
    }
    if (cache->sequences > 65535 || cache->kv_heads > 4096 || tokens > (1 << 24) || heads > (1 << 16) ||
        cache->pages > 0x7FFFFFFF || cache->table_width > (1 << 26) / page * 16 || max_query > (1 << 24)) {
        record_error_text("too many sequences, heads, tokens or pages");
        return UE5M3_ERR_TOO_LARGE;
    }
    const int64_t strides[] = {cache->k_page_stride, cache->k_slot_stride, cache->k_head_stride, cache->v_page_stride,
                               cache->v_slot_stride, cache->v_head_stride, q_token_stride, q_head_stride,
                               new_k ? new_k_token_stride : 0, new_k ? new_k_head_stride : 0,
                               new_k ? new_v_token_stride : 0, new_k ? new_v_head_stride : 0};
    for (int64_t stride : strides)
        if (stride < 0 || stride % 8) return UE5M3_ERR_ALIGNMENT;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache->k_pages | (uintptr_t)cache->v_pages | (uintptr_t)new_k |
         (uintptr_t)new_v | (uintptr_t)workspace) % 16)
        return UE5M3_ERR_ALIGNMENT;
    const Plan plan = make_plan(tokens, cache->sequences, heads, cache->kv_heads, dim, max_query, max_kv);
    if (plan.workspace > 0 && (!workspace || workspace_bytes < plan.workspace)) return UE5M3_ERR_SCRATCH;

    Params p;
    p.q = reinterpret_cast<const __nv_bfloat16*>(q);
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.out = reinterpret_cast<__nv_bfloat16*>(out);
    p.page_table = cache->page_table;
    p.table_stride = cache->table_stride;
    p.kv_lengths = kv_lengths;
    p.query_starts = query_starts;
    p.v_pages = reinterpret_cast<const __nv_bfloat16*>(cache->v_pages);
    p.v_page = cache->v_page_stride;
    p.v_slot = cache->v_slot_stride;
    p.v_head = cache->v_head_stride;
    p.partial = reinterpret_cast<float*>(workspace);
    p.status = status_dev;
    p.sequences = (int)cache->sequences;
    p.tokens = (int)tokens;
    p.heads = (int)heads;
    p.kv_heads = (int)cache->kv_heads;
    p.group = (int)(heads / cache->kv_heads);
    p.table_width = (int)cache->table_width;
    p.pages = (int)cache->pages;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page) ++p.page_shift;
    p.chunk = plan.chunk;
    p.splits = plan.splits;
    p.zero_tail = zero_tail != 0;
    p.scale_log2 = scale * 1.4426950408889634f;

    CUtensorMap k_map, v_map;
    const int box = page < kKeys ? (int)page : kKeys;
    int status = encode_pages(&k_map, cache->k_pages, *cache, cache->k_page_stride, cache->k_slot_stride,
                              cache->k_head_stride, (int)dim, box);
    if (status == UE5M3_OK)
        status = encode_pages(&v_map, cache->v_pages, *cache, cache->v_page_stride, cache->v_slot_stride,
                              cache->v_head_stride, (int)dim, box);
    if (status != UE5M3_OK) return status;
    AppendParams a = {};
    if (new_k) {
        a.k = reinterpret_cast<const __nv_bfloat16*>(new_k);
        a.v = reinterpret_cast<const __nv_bfloat16*>(new_v);
        a.k_token = new_k_token_stride;
        a.k_head = new_k_head_stride;
        a.v_token = new_v_token_stride;
        a.v_head = new_v_head_stride;
        a.k_pages = reinterpret_cast<__nv_bfloat16*>(cache->k_pages);
        a.v_pages = reinterpret_cast<__nv_bfloat16*>(cache->v_pages);
        a.k_page = cache->k_page_stride;
        a.k_slot = cache->k_slot_stride;
        a.k_page_head = cache->k_head_stride;
        a.v_page = cache->v_page_stride;
        a.v_slot = cache->v_slot_stride;
        a.v_page_head = cache->v_head_stride;
    }
    cudaStream_t s = (cudaStream_t)stream;
    return dim == 64 ? launch<64>(p, plan, k_map, v_map, a, max_query, s)
                     : launch<128>(p, plan, k_map, v_map, a, max_query, s);
}
