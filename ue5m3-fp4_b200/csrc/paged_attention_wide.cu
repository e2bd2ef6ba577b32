// Attention of a chunk of new tokens over a paged key/value cache: the kernel for many rows (prompt
// chunks).
//
// What bounds it: the tensor cores (4 * head_dim flops per row and visible key) and, nearly as much,
// the exponentials.  One CTA owns 256 rows of a key/value head (its query heads side by side, see
// paged_attention.cuh) as two tiles of 128, so that one tile's softmax runs while the other's
// products do.  Per 128 keys: S = Q K^T (tcgen05.mma, both operands in shared memory) into TMEM; a
// warpgroup per tile, one thread per row, reads S, keeps the running maximum and sum in fp32 and
// writes the probabilities as bf16 over S; O += P V with P read from TMEM and V [keys][channels]
// as it lies in the cache (the N-major operand), O in fp32 in TMEM.
//
// TMEM: S/P of the two tiles 128 columns each, O head_dim columns each.  The output is rescaled
// only when a row's maximum has grown by more than 2^8 since the last time (probabilities then stay
// below 2^8, which bf16 and the fp32 sums hold as well as any), so that TMEM is hardly ever read
// and written between products.
//
// Warps: 0 TMA (keys and values page by page into two stages of 128 keys each), 1 MMA issue and
// TMEM, 2 and 3 the values of keys that not every row sees (cleared, or kept finite, before a product
// meets them), 4..11 the softmax of the two tiles (TMEM lanes by warp % 4).
//
// Measured: 2048 tokens of 8192 keys, 32 heads over 4 key/value heads of 128: 236 us, 1020 TFLOP/s of
// 1649.  Per 2 x 128 x 128 scores an SM is active for 3800 cycles, in 2070 of which its tensor pipe is: with
// head_dim 128 TMEM has room for one whole S per tile beside the outputs, so a tile's products wait for
// its softmax and only the other tile's hide it (head_dim 64 leaves 128 columns unused).  Scores by the
// issuing warp's additions to constant descriptors: 300 -> 243 us; probabilities handed over in halves and
// keys' stages released by the warps that see the scores: 236.  Slower, each: 64 keys per step 306, a
// polynomial in place of some ex2, scores read from TMEM twice.
//
// A probability is rounded to bf16 for its product, its row's sum takes it unrounded: with the output's
// own rounding the relative error is 0.0023 where one rounding leaves 0.0017.  Summing the rounded ones
// instead gives 0.0022 and takes 287 us in place of 236 (the softmax's registers no longer suffice).
#include <math.h>

#include "abi_common.cuh"
#include "paged_attention.cuh"
#include "tcgen05_ptx.cuh"

namespace ue5m3 {
namespace paged {

constexpr int kWideKeys = 128;   // keys of a stage
constexpr int kWideStages = 2;
constexpr int kWideThreads = 384;
constexpr float kRescale = 8.0f;  // log2 of the growth of a maximum that is left in the probabilities
constexpr int kSiteWide = 0x60;
constexpr int kProducerRegisters = 88, kSoftmaxRegisters = 208;  // 128 * 88 + 256 * 208 <= 384 * 168

template <int kDim>
struct WideShared {
    static constexpr int kSlabs = kDim / 64;
    static constexpr int kTileBytes = 128 * kDim * 2;  // 128 rows or keys: kSlabs x [128][128 bytes], swizzled
    static constexpr int kQ = 0;
    static constexpr int kK = 2 * kTileBytes;
    static constexpr int kV = kK + kWideStages * kTileBytes;
    static constexpr int kBarriers = kV + kWideStages * kTileBytes;
    static constexpr int kBytes = kBarriers + 2048 + 1024;
};

struct WideBarriers {
    unsigned long long k_full[kWideStages], k_empty[kWideStages], v_full[kWideStages];
    unsigned long long q_ready, s_full[2], p_half[2], p_ready[2], o_done[2], drained;
    unsigned long long v_there[kWideStages], v_settled[kWideStages];  // per stage: its next use waits for this one's
    uint32_t tmem;
    int abort_flag, bad;
    int odd_count;             // keys with values that are not finite and that not every row sees
    int odd_keys[kWideRows];
};

// Instruction descriptor for kind::f16, D = F32, A = B = BF16; b_rows: B is [k][n] in memory
__host__ __device__ constexpr uint32_t wide_idesc(int m, int n, bool b_rows) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// B operand [k][n], n contiguous: 64-channel slabs of [keys][128 bytes], 128-byte swizzle; slabs
// are kWideKeys * 128 bytes apart, groups of eight keys 1024 bytes
__device__ __forceinline__ uint64_t desc_rows(uint32_t address) {
    uint64_t desc = 0;
    desc |= (uint64_t)((address & 0x3FFFFu) >> 4);
    desc |= (uint64_t)((kWideKeys * 128) >> 4) << 16;
    desc |= (uint64_t)(1024 >> 4) << 32;
    desc |= (uint64_t)1 << 46;
    desc |= (uint64_t)2 << 61;
    return desc;
}

__device__ __forceinline__ void tmem_store_16(uint32_t address, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Waits for this thread's TMEM loads.  The registers pass through the statement, so that nothing
// that reads them can be moved before the wait.
template <int kCount>
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[kCount]) {
    ptx::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < kCount; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ void tmem_load_16(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address)
        : "memory");
}

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A row of V in its tile whose key not every row sees: behind the last key it is cleared; otherwise
// values that are not finite become zero, and the key is noted.
template <int kDim>
__device__ void settle_values(unsigned char* v, int key, int key_end, WideBarriers& bar) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i) {
        uint4* piece = reinterpret_cast<uint4*>(v + (i / 8) * kWideKeys * 128 + (i & 7) * 16);
        if (key >= key_end) {
            *piece = make_uint4(0, 0, 0, 0);
        } else if (odd_piece(*piece)) {
            odd = true;
            uint32_t* w = reinterpret_cast<uint32_t*>(piece);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if ((w[e] & 0x7F80u) == 0x7F80u) w[e] &= 0xFFFF0000u;
                if ((w[e] & 0x7F800000u) == 0x7F800000u) w[e] &= 0xFFFFu;
            }
        }
    }
    if (odd) bar.odd_keys[atomicAdd(&bar.odd_count, 1) % kWideRows] = key;
}

// one row tile's work
struct Job {
    int row0, limit, key_begin, key_end, tiles, splits;
    bool mine;  // this CTA's split has keys of it, or it is the one that writes the zeros of rows without any
};

// later row tiles see more keys: they come first
__device__ __forceinline__ Job job_of(const Params& p, const Sequence& s, int rows, int at) {
    Job job;
    job.row0 = ((rows + kWideRows - 1) / kWideRows - 1 - at) * kWideRows;
    job.limit = visible_keys(p, s, job.row0, kWideRows);
    const int all = (job.limit + kKeys - 1) / kKeys;  // in units of the split, 64 keys
    const int chunk = split_chunk(p, all);
    job.splits = (all + chunk - 1) / chunk;
    const int first = blockIdx.x * chunk;
    job.mine = first < all || blockIdx.x == 0;
    job.key_begin = first * kKeys;
    job.key_end = min(job.limit, (first + chunk) * kKeys);
    job.tiles = (job.key_end - job.key_begin + kWideKeys - 1) / kWideKeys;
    return job;
}

template <int kDim>
__global__ void __launch_bounds__(kWideThreads, 1)
    attention_wide_kernel(const Params p, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
    using Shared = WideShared<kDim>;
    constexpr int kSlabs = Shared::kSlabs, kTileBytes = Shared::kTileBytes;
    extern __shared__ unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    WideBarriers& bar = *reinterpret_cast<WideBarriers*>(smem + Shared::kBarriers);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z;
    const int row_tiles = gridDim.y / p.kv_heads;
    const int head = blockIdx.y % p.kv_heads;  // the row tiles that see most keys start first, of all heads
    const Sequence s = sequence_of(p, b);
    if (p.zero_tail)
        zero_tail_rows(p, ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kWideThreads + threadIdx.x,
                       (int64_t)gridDim.x * gridDim.y * gridDim.z * kWideThreads, kDim);
    const int rows = s.queries * p.group;
    if (rows == 0) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kWideStages; ++i) {
            ptx::mbar_init(&bar.k_full[i], 1);
            ptx::mbar_init(&bar.k_empty[i], 4);
            ptx::mbar_init(&bar.v_full[i], 1);
            ptx::mbar_init(&bar.v_there[i], 1);
            ptx::mbar_init(&bar.v_settled[i], 2);
        }
        ptx::mbar_init(&bar.q_ready, 256);
        ptx::mbar_init(&bar.drained, 1);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&bar.s_full[i], 1);
            ptx::mbar_init(&bar.p_half[i], 4);
            ptx::mbar_init(&bar.p_ready[i], 4);
            ptx::mbar_init(&bar.o_done[i], 1);
        }
        bar.odd_count = 0;
        bar.abort_flag = p.status && *((volatile int*)p.status) != 0;  // a recorded failure: no work, NaN
        ptx::mbar_fence_init();
    }
    if (warp == 1) ptx::tmem_alloc(&bar.tmem, 512);
    launch_dependents();
    wait_for_launcher();  // the new keys and values are in their pages ...
    asm volatile("fence.proxy.async;" ::: "memory");  // ... and TMA sees them
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::tcgen05_fence_after();
    const uint32_t tmem = bar.tmem;
    constexpr uint32_t kS = 0, kO = 256;  // columns: S of tile t at 128 t, O at 256 + kDim t
    int stage_count = 0;   // key stages used so far (every role counts alike); also the per-tile barriers' phases
    int list = 0;          // row tiles done so far
    int finished = 0;      // row tiles with keys done so far
    uint32_t settled = 0;  // per stage, the parity of the tiles of V that needed settling
    // between two row tiles; true when a wait gave up, here or in an earlier launch
    auto begin = [&]() {
        __syncthreads();
        if (threadIdx.x == 0) bar.bad = s.cut;
        __syncthreads();
        return *((volatile int*)&bar.abort_flag) != 0;
    };
    // Seldom: the noted keys' values that are not finite, added to the finished rows that see them (their
    // weights are positive): to the output, or, where the keys are split, to the partial rows.  Warp 2.
    auto add_odd_values = [&](const Job& job) {
        const int count = min(*((volatile int*)&bar.odd_count), kWideRows);
        for (int i = lane; i < count * min(kWideRows, rows - job.row0); i += 32) {
            const int key = bar.odd_keys[i % count], row = job.row0 + i / count, token = row / p.group;
            const int page = key <= s.keys - s.queries + token ? page_of(p, b, key) : -1;
            if (page < 0) continue;
            const __nv_bfloat16* v = p.v_pages + page * p.v_page + (key & ((1 << p.page_shift) - 1)) * p.v_slot + head * p.v_head;
            const int64_t at = (int64_t)(s.first + token) * p.heads + head * p.group + row % p.group;
            for (int d = 0; d < kDim; ++d) {
                const float value = __bfloat162float(v[d]);
                if (fabsf(value) <= 3.4e38f) continue;
                if (job.splits <= 1)
                    atomicAdd(p.out + at * kDim + d, v[d]);  // finite + inf, inf + inf, inf - inf: the same in any order
                else
                    atomicAdd(p.partial + (at * p.splits + blockIdx.x) * kDim + d, value);
            }
        }
        __syncwarp();
        if (lane == 0) bar.odd_count = 0;
    };
    if (warp < 4) {
        // a row's 128 scores live in registers: what these roles do not need goes to the softmax
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegisters));
        for (int at = blockIdx.y / p.kv_heads; at * kWideRows < rows; at += row_tiles) {
            const Job job = job_of(p, s, rows, at);
            if (!job.mine) continue;
            const int key_begin = job.key_begin, key_end = job.key_end, tiles = job.tiles;
            const int all_see = visible_keys(p, s, job.row0, 1);  // keys that every row sees
            const int settle_from = min(all_see, key_end);        // tiles with keys from here on are settled
            const bool dead = begin();
            if (warp == 0) {
                if (!dead) {
                    const int box = min(kKeys, 1 << p.page_shift), boxes = kWideKeys / box;
                    int j = 0;
                    for (; j < tiles; ++j) {
                        const int n = stage_count + j, stage = n % kWideStages, parity = (n / kWideStages) & 1;
                        const int key = key_begin + j * kWideKeys + lane * box;
                        const bool wanted = lane < boxes && key < key_end;
                        const int page = wanted ? page_of(p, b, key) : -1;
                        if (wanted && page < 0) bar.bad = 1;
                        const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, page >= 0)) * box * kDim * 2;
                        const int slot = key & ((1 << p.page_shift) - 1);
                        unsigned char* to = smem + Shared::kK + stage * kTileBytes + lane * box * 128;
                        if (n >= kWideStages &&
                            !warp_wait(&bar.k_empty[stage], parity ^ 1, &bar.abort_flag, p.status, kSiteWide, n))
                            break;
                        if (lane == 0) ptx::mbar_arrive_expect_tx(&bar.k_full[stage], bytes);
                        __syncwarp();
                        if (page >= 0)
                            for (int i = 0; i < kSlabs; ++i)
                                tma_load_4d(to + i * kWideKeys * 128, &k_map, &bar.k_full[stage], i * 64, head, slot, page);
                        // the scores of tile n - 1 are issued behind the products with the values of tile n - 2
                        if (n >= kWideStages && !warp_wait(&bar.k_empty[(n - 1) % kWideStages], ((n - 1) / kWideStages) & 1,
                                                           &bar.abort_flag, p.status, kSiteWide + 1, n)) {
                            // the copy of K of this tile lands before its memory is given up
                            for (int spin = 0; spin < 1000000 && !ptx::mbar_try_wait(&bar.k_full[stage], parity);) ++spin;
                            break;
                        }
                        if (lane == 0) ptx::mbar_arrive_expect_tx(&bar.v_full[stage], bytes);
                        __syncwarp();
                        to += Shared::kV - Shared::kK;
                        if (page >= 0)
                            for (int i = 0; i < kSlabs; ++i)
                                tma_load_4d(to + i * kWideKeys * 128, &v_map, &bar.v_full[stage], i * 64, head, slot, page);
                        if (key_begin + (j + 1) * kWideKeys > settle_from) {
                            // warps 2 and 3 follow no other tiles and could not tell one phase of v_full from the next
                            if (!warp_wait(&bar.v_full[stage], parity, &bar.abort_flag, p.status, kSiteWide + 12, n)) {
                                ++j;
                                break;
                            }
                            if (lane == 0) ptx::mbar_arrive(&bar.v_there[stage]);
                        }
                    }
                    if (*((volatile int*)&bar.abort_flag))
                        for (int i = max(0, stage_count + j - kWideStages); i < stage_count + j; ++i)
                            for (int spin = 0; spin < 1000000 && !(ptx::mbar_try_wait(&bar.k_full[i % kWideStages], (i / kWideStages) & 1) &&
                                                                   ptx::mbar_try_wait(&bar.v_full[i % kWideStages], (i / kWideStages) & 1));)
                                ++spin;
                }
            } else if (warp == 1) {
                constexpr uint32_t kIdescS = wide_idesc(128, kWideKeys, false), kIdescO = wide_idesc(128, kDim, true);
                // descriptors differ by constants (in units of 16 bytes), so that an issue costs an addition
                const uint32_t base = ptx::smem_u32(smem);
                const uint64_t q_desc = ptx::smem_desc_sw128(base + Shared::kQ), k_desc = ptx::smem_desc_sw128(base + Shared::kK),
                               v_desc = desc_rows(base + Shared::kV);
                auto scores = [&](int t, int stage) {
                    const uint64_t q = q_desc + t * (kTileBytes / 16), k = k_desc + stage * (kTileBytes / 16);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int i = 0; i < kDim / 16; ++i) {
                            const int off = ((i / 4) * kWideKeys * 128 + (i % 4) * 32) / 16;
                            umma_ss(tmem + kS + 128 * t, q + off, k + off, kIdescS, i > 0);
                        }
                        ptx::umma_commit(&bar.s_full[t]);
                    }
                    __syncwarp();
                };
                auto values = [&](int t, int stage, int half, bool accumulate, bool last) {
                    const uint64_t v = v_desc + stage * (kTileBytes / 16) + half * (kTileBytes / 32 / kSlabs);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int k = 0; k < kWideKeys / 32; ++k) {
                            umma_ts(tmem + kO + kDim * t, tmem + kS + 128 * t + 8 * (half * (kWideKeys / 32) + k), v + k * 128,
                                    kIdescO, accumulate || k > 0);
                        }
                        if (last && half == 1) ptx::umma_commit(&bar.o_done[t]);
                    }
                    __syncwarp();
                };
                auto wait = [&](unsigned long long* which, uint32_t parity, int site) {
                    const bool ok = warp_wait(which, parity, &bar.abort_flag, p.status, kSiteWide + site, stage_count);
                    ptx::tcgen05_fence_after();
                    return ok;
                };
                bool ok = !dead && tiles > 0 && wait(&bar.q_ready, list & 1, 2);
                ok = ok && wait(&bar.k_full[stage_count % kWideStages], (stage_count / kWideStages) & 1, 3);
                if (ok) {
                    scores(0, stage_count % kWideStages);
                    scores(1, stage_count % kWideStages);
                }
                for (int j = 0; ok && j < tiles; ++j) {
                    const int n = stage_count + j, stage = n % kWideStages, next = (n + 1) % kWideStages;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok) break;
                        ok = wait(&bar.p_half[t], n & 1, 4);
                        if (ok && t == 0) {
                            ok = wait(&bar.v_full[stage], (n / kWideStages) & 1, 5);
                            if (ok && key_begin + (j + 1) * kWideKeys > settle_from) {
                                ok = wait(&bar.v_settled[stage], settled >> stage & 1, 9);
                                settled ^= 1u << stage;
                            }
                        }
                        if (!ok) break;
                        values(t, stage, 0, j > 0, false);
                        ok = wait(&bar.p_ready[t], n & 1, 7);
                        if (!ok) break;
                        values(t, stage, 1, true, j == tiles - 1);
                        if (j + 1 < tiles) {
                            if (t == 0) ok = wait(&bar.k_full[next], ((n + 1) / kWideStages) & 1, 6);
                            if (ok) scores(t, next);
                        }
                    }
                }
            } else if (!dead) {
                // Warps 2 and 3: values of keys that no row sees, or not every one, must not meet the others' zero
                // probabilities where they are not finite.  The former are cleared; of the latter those that
                // are not finite, which the rows that see the key get in the end.
                for (int j = 0; j < tiles; ++j) {
                    const int key0 = key_begin + j * kWideKeys, stage = (stage_count + j) % kWideStages;
                    if (key0 + kWideKeys <= settle_from) continue;
                    if (!warp_wait(&bar.v_there[stage], settled >> stage & 1, &bar.abort_flag, p.status, kSiteWide + 10, j)) break;
                    settled ^= 1u << stage;
                    for (int r = (warp - 2) * 32 + lane; r < kWideKeys; r += 64)
                        if (key0 + r >= all_see || key0 + r >= key_end)
                            settle_values<kDim>(smem + Shared::kV + stage * kTileBytes + r * 128, key0 + r, key_end, bar);
                    asm volatile("fence.proxy.async;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&bar.v_settled[stage]);
                }
            }
            stage_count += tiles;
            ++list;
            __syncthreads();  // the rows are written
            if (warp == 2 && *((volatile int*)&bar.odd_count) != 0) add_odd_values(job);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        for (int at = blockIdx.y / p.kv_heads; at * kWideRows < rows; at += row_tiles) {
            const Job job = job_of(p, s, rows, at);
            if (!job.mine) continue;
            const int row0 = job.row0, key_begin = job.key_begin, tiles = job.tiles, splits = job.splits;
            const bool dead = begin();
            const int t = (warp - 4) / 4, r = (warp % 4) * 32 + lane;  // tile, row in it
            const uint32_t lanes = tmem + ((uint32_t)((warp % 4) * 32) << 16);
            const int row = row0 + t * 128 + r;
            const int token = row / p.group;
            const bool present = row < rows;
            const int last_key = present ? s.keys - s.queries + token : -1;
            const int fewest = visible_keys(p, s, min(row0 + t * 128, rows - 1), 1);  // of the tile's rows
            float top = -INFINITY, sum = 0.0f;
            if (!dead) {
                // this thread's row of Q into the swizzled tile
                const uint4* source = reinterpret_cast<const uint4*>(
                    p.q + (int64_t)(s.first + token) * p.q_token + (int64_t)(head * p.group + row % p.group) * p.q_head);
                unsigned char* q = smem + Shared::kQ + t * kTileBytes + r * 128;
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i)
                    *reinterpret_cast<uint4*>(q + (i / 8) * 128 * 128 + (((i & 7) ^ (r & 7)) << 4)) =
                        present ? source[i] : make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async;" ::: "memory");
                ptx::mbar_arrive(&bar.q_ready);
            }
            bool ok = !dead;
            for (int j = 0; ok && j < tiles; ++j) {
                const int key0 = key_begin + j * kWideKeys;
                const uint32_t parity = (stage_count + j) & 1;
                ok = warp_wait(&bar.s_full[t], parity, &bar.abort_flag, p.status, kSiteWide + 8, j);
                if (!ok) break;
                ptx::tcgen05_fence_after();
                // the keys' stage is free when both tiles' scores are; a commit for it would cost the issuing warp
                if (t == 1 && lane == 0) ptx::mbar_arrive(&bar.k_empty[(stage_count + j) % kWideStages]);
                const bool masked = key0 + kWideKeys > fewest;
                uint32_t x[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) ptx::tmem_load_32_async(lanes + kS + 128 * t + 32 * i, x[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_loaded(x[i]);
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 128; ++e)
                        if (key0 + e > last_key) x[e / 32][e % 32] = 0xFF800000u;
                }
                float most[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    most[i] = fmaxf(__uint_as_float(x[i][0]), __uint_as_float(x[i][1]));
#pragma unroll
                    for (int e = 2; e < 32; e += 2)
                        most[i] = max3(most[i], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
                }
                const float now = max3(fmaxf(most[0], most[1]), most[2], most[3]) * p.scale_log2;
                if (__any_sync(0xFFFFFFFFu, now > top + kRescale || (top == -INFINITY && now > top))) {
                    // the maximum moves; what has been summed so far fades
                    const float moved = fmaxf(top, now);
                    const float fade = moved == -INFINITY ? 1.0f : exp2_approx(top - moved);
                    sum *= fade;
                    top = moved;
                    if (j > 0) {  // the scores' arrival tells that the products before them are done
#pragma unroll 1
                        for (int i = 0; i < kDim / 16; ++i) {
                            uint32_t o[16];
                            tmem_load_16(lanes + kO + kDim * t + 16 * i, o);
                            tmem_loaded(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                            tmem_store_16(lanes + kO + kDim * t + 16 * i, o);
                        }
                    }
                }
                const float base = top == -INFINITY ? 0.0f : top;
                const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), base2 = pack2(-base, -base);
                uint64_t sums[4] = {0, 0, 0, 0};
                auto probabilities = [&]() {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const uint64_t y = fma2(pack2(__uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1])), scale2, base2);
                            float lo, hi;
                            unpack2(y, lo, hi);
                            lo = exp2_approx(lo);
                            hi = exp2_approx(hi);
                            sums[(e / 2) % 4] = add2(sums[(e / 2) % 4], pack2(lo, hi));
                            packed[e / 2] = pack_bf16(lo, hi);
                        }
                        tmem_store_16(lanes + kS + 128 * t + 16 * i, packed);
                        if (i & 1) {  // the product with the first 64 keys starts while the others are computed
                            tmem_wait_st();
                            ptx::tcgen05_fence_before();
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(i == 1 ? &bar.p_half[t] : &bar.p_ready[t]);
                        }
                    }
                };
                // written twice: the compiler's schedule of the common case is better for it (232 against 260 us)
                if (masked)
                    probabilities();
                else
                    probabilities();
                float lo, hi;
                unpack2(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])), lo, hi);
                sum += lo + hi;
            }
            if (ok && tiles > 0)
                ok = warp_wait(&bar.o_done[t], finished++ & 1, &bar.abort_flag, p.status, kSiteWide + 11, 0);
            ptx::tcgen05_fence_after();
            __syncwarp();
            const bool failed = !ok || *((volatile int*)&bar.abort_flag) || *((volatile int*)&bar.bad);
            const int64_t out_at = (int64_t)(s.first + token) * p.heads + head * p.group + row % p.group;
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
            for (int i = 0; i < kDim / 32; ++i) {
                uint32_t x[32];
                __syncwarp();
                if (tiles > 0 && !dead) {
                    ptx::tmem_load_32_async(lanes + kO + kDim * t + 32 * i, x);
                    tmem_loaded(x);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float v = tiles > 0 && !dead ? __uint_as_float(x[e]) : 0.0f;
                    if (sum == 0.0f) v = 0.0f;
                    if (failed) v = __uint_as_float(0x7FC00000u);
                    x[e] = __float_as_uint(v);
                }
                if (present && splits <= 1) {
                    uint4* to = reinterpret_cast<uint4*>(p.out + out_at * kDim + 32 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = pack_bf16(__uint_as_float(x[8 * e + 2 * k]) * inverse,
                                             __uint_as_float(x[8 * e + 2 * k + 1]) * inverse);
                        to[e] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (splits > 1) {
                    // a thread has a row, a store wants neighbouring pieces: through this tile's part of Q, which
                    // is read no more
                    unsigned char* turn = smem + Shared::kQ + t * kTileBytes + (warp % 4) * 4096;
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *reinterpret_cast<uint4*>(turn + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                            make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int from = e * 4 + lane / 8, piece = lane % 8;
                        const int64_t row_at = __shfl_sync(0xFFFFFFFFu, present ? out_at : -1, from);
                        if (row_at >= 0)
                            *reinterpret_cast<uint4*>(p.partial + (row_at * p.splits + blockIdx.x) * kDim + 32 * i + 4 * piece) =
                                *reinterpret_cast<const uint4*>(turn + from * 128 + ((piece ^ (from & 7)) << 4));
                    }
                }
            }
            if (splits > 1 && present) {
                float* stats = p.partial + (int64_t)p.tokens * p.heads * p.splits * kDim + (out_at * p.splits + blockIdx.x) * 2;
                stats[0] = failed ? 0.0f : top;
                stats[1] = failed ? __uint_as_float(0x7FC00000u) : sum;
            }
            ptx::tcgen05_fence_before();
            stage_count += tiles;
            __syncthreads();
        }
    }
    __syncthreads();
    if (warp == 1) {
        if (*((volatile int*)&bar.abort_flag)) {
            // products in flight end before their memory is given up
            if (ptx::elect_one()) ptx::umma_commit(&bar.drained);
            __syncwarp();
            for (int spin = 0; spin < 1000000 && !ptx::mbar_try_wait(&bar.drained, 0);) ++spin;
            __syncwarp();
        }
        ptx::tcgen05_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

template <int kDim>
static int launch_wide_dim(const Params& p, dim3 grid, const CUtensorMap& k_map, const CUtensorMap& v_map, bool early,
                           cudaStream_t stream) {
    cudaError_t error = allow_shared<attention_wide_kernel<kDim>>(WideShared<kDim>::kBytes);
    if (error == cudaSuccess)
        error = launch_after(attention_wide_kernel<kDim>, grid, kWideThreads, WideShared<kDim>::kBytes, stream, early, p, k_map,
                             v_map);
    return record_cuda_error(error);
}

int launch_wide(const Params& p, int head_dim, dim3 grid, const CUtensorMap& k_map, const CUtensorMap& v_map, bool early,
                cudaStream_t stream) {
    return head_dim == 64 ? launch_wide_dim<64>(p, grid, k_map, v_map, early, stream)
                          : launch_wide_dim<128>(p, grid, k_map, v_map, early, stream);
}

}  // namespace paged
}  // namespace ue5m3
