// The next token of every row of logits from one given uniform number per row:
//   w_i = exp((l_i - max l) / T);   kept: the top_k largest, of these the shortest descending prefix
//   whose weight reaches top_p of theirs, of these the tokens with w_i >= min_p;
//   token = the first kept i, in vocabulary order, with w_0 + ... + w_i > u * (sum of the kept).
// Equal logits rank by their index, lowest first.
//
// Arithmetic.  A token is chosen by comparing long sums with a border, so the sums are exact: the
// weight is computed in fp64 and rounded once to a multiple of 2^-44, and all sums are integers.
// No order of additions, split or atomic can change a result.  An element's rank is the 64-bit
// integer (logit in integer order, complement of its index), which no two elements share; top-k
// and top-p each end as one threshold on it.
//
// What bounds it: a batch of rows, one fp64 exponential per logit that a sum needs, then reading the
// logits; a single row, the latency of its steps.  A cluster of up to eight CTAs holds a row in
// shared memory, so that it is read from memory once however many steps follow.  A step of a
// threshold search is a histogram of 512 bins over the row, summed over the cluster through
// distributed shared memory by every CTA for itself (one cluster barrier per step).  The first
// step's bins are linear in (max - l) / T, which spreads real logits (bins of the integer order
// would put a fifth of a row into one of them); what lies in the last, open bin is counted in
// registers.  Where the first step leaves at most 256 elements that can be kept (top-k of a few
// hundred, a peaked nucleus), these are gathered and the rest happens among them in one CTA.
// Otherwise the elements of the bin that holds the threshold are ranked against one another, or the
// search goes on inside it with bins of the 64-bit rank (many equal logits).
//
// Measured (fp32): one row of 131072, top-k and top-p: 13.5 us, the steps of eight CTAs that wait
// for one another at four cluster barriers; top-p alone 27 us; 64 rows of 131072 with top-p alone:
// 84 us, against 5 us for the bytes and 6.5 us for the exponentials at the rate of the fp64 pipe: two
// CTAs fit on an SM, so the 512 take almost two turns of weights, their atomics (32 logits a thread) and
// steps that wait.  Of its active cycles it issues in 41 % of the slots, the fp64 pipe is busy in 9 %;
// barriers are the largest stall.  Weights of the nucleus alone in the last step, bins summed once per CTA
// before the others read them, and ranking by all threads of the cluster took it there from 111.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "abi_common.cuh"

namespace ue5m3 {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;          // one bin per thread in the scan over bins
constexpr int kCandidates = 1024;        // elements that are ranked against one another
constexpr int kFew = 256;                // ... in one CTA, to the end (64 rows of 32000, top-k 400: 59 us; 512: 77)
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxVocabulary = 1 << 18;
constexpr float kBinsPerUnit = 32.0f;    // first step: bins of (max - l) / T, the last one open
constexpr double kOne = 17592186044416.0;  // 2^44

struct Params {
    const void* logits;
    int64_t ld;
    const float* uniforms;
    const float* temperature_dev;
    const int* top_k_dev;
    const float* top_p_dev;
    const float* min_p_dev;
    float temperature;
    int top_k;
    float top_p, min_p;
    long long* tokens;
    float* logprobs;
    int vocabulary;
    int slice;  // elements of a row per CTA of the cluster
    int bf16, vector;
};

struct alignas(16) Shared {
    double power[8];             // 2^(j / 8)
    uint32_t hist[4][kBins];  // [count, weight bits 0..16, 17..33, 34..44]: 2^15 summands fit
    uint64_t bin_weight[2][kBins];  // a step's bins of this CTA for the others, which may still read those of the
    uint32_t bin_number[2][kBins];  // step before
    uint64_t mine[kCandidates];  // this CTA's candidates
    uint64_t all[kCandidates];
    uint64_t weight[kCandidates];
    uint64_t warp_sum[kWarps];
    uint64_t cta_sum;
    uint64_t found, found_before;
    uint64_t low, high;          // bounds of the ranks in a bin (this CTA's)
    float warp_top[kWarps], cta_top;
    uint32_t first_top, count;
    uint32_t found_bin, found_count, found_through;
    uint32_t warp_number[kWarps];
};

// logits in integer order: a larger logit has a larger key
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint64_t rank_of(uint32_t key, uint32_t index) {
    return (uint64_t)key << 32 | (0xFFFFFFFFu - index);
}

// share * total for 0 <= share < 1, rounded down or up to an integer, exactly
__device__ __forceinline__ uint64_t share_of(float share, uint64_t total, bool up) {
    const uint32_t bits = __float_as_uint(share);
    const uint32_t field = bits >> 23 & 0xFF;
    const uint64_t mantissa = (bits & 0x7FFFFFu) | (field ? 0x800000u : 0u);
    const int shift = 150 - (field ? (int)field : 1);  // share = mantissa * 2^-shift, shift >= 24
    const uint64_t low = total * mantissa, high = __umul64hi(total, mantissa);
    uint64_t whole, rest;
    if (shift < 64) {
        whole = high << (64 - shift) | low >> shift;
        rest = low << (64 - shift);
    } else {
        const int cut = min(shift - 64, 63);  // high is below 2^23
        whole = high >> cut;
        rest = low | (high & (((uint64_t)1 << cut) - 1));
    }
    return whole + (up && rest ? 1 : 0);
}

struct Row {
    float top;            // the largest logit
    double inverse;       // 1 / T
    float bin_scale;      // kBinsPerUnit / T, finite
    const double* power;  // 2^(j / 8) in shared memory
};

__device__ __forceinline__ double exponent_of(const Row& row, float v) {
    const double z = ((double)v - (double)row.top) * row.inverse;
    return v == row.top ? 0.0 : z;  // also where both are infinite
}

// 2^44 exp(z), z <= 0, to the nearest integer.  z = k ln(2) / 8 + r: a power of two, a table of eight
// and Taylor's polynomial of degree 7, whose remainder on |r| <= ln(2) / 16 is below 2^-51 of the
// value (ln(2) / 8 is rounded, which k <= 361 makes less than 2^-48).  Adding 1.5 * 2^52 leaves the
// nearest integer in the low bits.
__device__ __forceinline__ uint64_t weight_of(const Row& row, float v) {
    const double z = exponent_of(row, v);
    constexpr double kMagic = 6755399441055744.0;
    const double shifted = fma(z, 8.0 * 1.4426950408889634, kMagic);
    const int k = __double2loint(shifted);
    const double r = fma(shifted - kMagic, -0.6931471805599453 / 8.0, z);
    double e = 1.0 / 5040.0;
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0) * row.power[k & 7];
    e = __hiloint2double(__double2hiint(e) + (((k >> 3) + 44) << 20), __double2loint(e)) + kMagic;
    const uint64_t w = (uint64_t)__double_as_longlong(e) & (((uint64_t)1 << 51) - 1);
    return z > -31.2 ? w : 0;  // below half a unit, or masked
}

__device__ __forceinline__ uint32_t first_bin(const Row& row, float v) {
    // monotone in v, as each step rounds monotonely; 2^23 leaves the nearest integer in the low bits
    const float bin = fminf((row.top - v) * row.bin_scale, (float)(kBins - 1)) + 8388608.0f;
    return v == row.top ? 0 : __float_as_uint(bin) & (kBins - 1);
}

// f(four neighbouring logits, place of the first in the slice); the slice is filled up to whole
// quadruples with minus infinity.  What f does to the four is written without branches where it is
// done to all of a row: their latencies would add up.
template <typename Function>
__device__ __forceinline__ void for_each_four(const float* data, int count, Function f) {
    for (int i = 4 * threadIdx.x; i < count; i += 4 * kThreads) {
        const float4 v = *reinterpret_cast<const float4*>(data + i);
        const float four[4] = {v.x, v.y, v.z, v.w};
        f(four, i);
    }
}

// f(logit, place in the slice) for the elements of a slice that are not masked
template <typename Function>
__device__ __forceinline__ void for_each(const float* data, int count, Function f) {
#pragma unroll 2
    for (int i = 4 * threadIdx.x; i < count; i += 4 * kThreads) {
        const float4 v = *reinterpret_cast<const float4*>(data + i);
        if (v.x != -INFINITY) f(v.x, i);
        if (v.y != -INFINITY) f(v.y, i + 1);
        if (v.z != -INFINITY) f(v.z, i + 2);
        if (v.w != -INFINITY) f(v.w, i + 3);
    }
}

// f(0) ... f(kMaxCluster - 1), unrolled: reads of other CTAs' memory are in flight together
template <typename Function>
__device__ __forceinline__ void for_each_cta(Function f) {
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) f(r);
}

__device__ __forceinline__ uint64_t warp_total(uint64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}

__device__ __forceinline__ uint64_t warp_running(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t from = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if ((int)(threadIdx.x & 31) >= d) v += from;
    }
    return v;
}

__device__ __forceinline__ void add_weight(uint32_t (*hist)[kBins], uint32_t bin, uint64_t w) {
    atomicAdd(&hist[1][bin], (uint32_t)(w & 0x1FFFF));
    atomicAdd(&hist[2][bin], (uint32_t)(w >> 17 & 0x1FFFF));
    if (w >> 34) atomicAdd(&hist[3][bin], (uint32_t)(w >> 34));  // within a factor of 1000 of the largest
}

// Where a histogram's running mass reaches `need`.
struct Found {
    uint64_t total;    // mass of all bins
    uint64_t before;   // mass of the bins above the one found
    uint32_t bin;
    uint32_t inside;   // elements in that bin
    uint32_t through;  // elements in it and the bins above
};

// The bins of all CTAs of the cluster, summed by each for itself (thread = bin), and the bin with
// which the running mass (number, or weight) reaches `need`; share > 0: need is that share of the
// total, rounded up.  Nothing is found where the total is below `need`.
template <bool kWeighted>
__device__ Found scan_bins(cg::cluster_group& cluster, Shared& s, int& buffer, uint64_t& need, float share) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    __syncthreads();
    s.bin_number[buffer][t] = s.hist[0][t];
    if (kWeighted) s.bin_weight[buffer][t] = (uint64_t)s.hist[1][t] + ((uint64_t)s.hist[2][t] << 17) + ((uint64_t)s.hist[3][t] << 34);
    cluster.sync();
    const int ctas = cluster.num_blocks();
    uint64_t weights[kMaxCluster];
    uint32_t numbers_of[kMaxCluster];
    for_each_cta([&](int r) {
        const Shared* other = cluster.map_shared_rank(&s, r < ctas ? r : 0);
        numbers_of[r] = other->bin_number[buffer][t];
        if (kWeighted) weights[r] = other->bin_weight[buffer][t];
    });
    uint64_t mass = 0;
    uint32_t number = 0;
    for_each_cta([&](int r) {
        if (r >= ctas) return;
        number += numbers_of[r];
        if (kWeighted) mass += weights[r];
    });
    buffer ^= 1;
    if (!kWeighted) mass = number;
    uint64_t running = warp_running(mass), numbers = kWeighted ? warp_running(number) : 0;
    if (lane == 31) {
        s.warp_sum[warp] = running;
        s.warp_number[warp] = (uint32_t)numbers;
    }
    __syncthreads();
    Found found;
    found.total = 0;
    uint64_t before = 0;
    uint32_t numbers_before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.warp_sum[w], numbers_before += s.warp_number[w];
        found.total += s.warp_sum[w];
    }
    running += before;
    if (share > 0.0f) need = share_of(share, found.total, true);
    if (running >= need && running - mass < need) {
        s.found_bin = t;
        s.found_before = running - mass;
        s.found_count = number;
        s.found_through = kWeighted ? numbers_before + (uint32_t)numbers : (uint32_t)running;
    }
    __syncthreads();
    found.bin = s.found_bin;
    found.before = s.found_before;
    found.inside = s.found_count;
    found.through = s.found_through;
    __syncthreads();
    return found;
}

__device__ __forceinline__ void clear_bins(Shared& s) {
    for (int i = 0; i < 4; ++i) s.hist[i][threadIdx.x] = 0;
    __syncthreads();
}

// The first step of a search among the elements with rank >= floor.
template <bool kWeighted>
__device__ Found first_step(cg::cluster_group& cluster, Shared& s, const float* data, int count, uint32_t base, const Row& row,
                            uint64_t floor, uint64_t& need, float share, int& buffer) {
    clear_bins(s);
    uint32_t(*hist)[kBins] = s.hist;
    uint64_t last_number = 0, last_weight = 0;
    for_each_four(data, count, [&](const float(&v)[4], int i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t bin = first_bin(row, v[e]);
            const uint64_t w = kWeighted ? weight_of(row, v[e]) : 1;
            bool in = kWeighted ? w != 0 : v[e] != -INFINITY;
            if (floor != 0) in = in && rank_of(key_of(v[e]), base + i + e) >= floor;
            const bool last = bin == kBins - 1;
            last_number += in && last;
            last_weight += in && last ? w : 0;
            if (in && !last) {
                atomicAdd(&hist[0][bin], 1u);
                if (kWeighted) add_weight(hist, bin, w);
            }
        }
    });
    last_number = warp_total(last_number);
    if (kWeighted) last_weight = warp_total(last_weight);
    if ((threadIdx.x & 31) == 0 && last_number) {
        atomicAdd(&hist[0][kBins - 1], (uint32_t)last_number);
        if (kWeighted) add_weight(hist, kBins - 1, last_weight);
    }
    return scan_bins<kWeighted>(cluster, s, buffer, need, share);
}

// Whether the first step counted an element that is not masked.  Weights of zero lie in its last bin,
// save at temperatures so small that the bins' scale is held back.
template <bool kWeighted>
__device__ __forceinline__ bool counted(const Row& row, float v) {
    return !kWeighted || weight_of(row, v) != 0;
}

// This CTA's elements that `look`, a glance at the logit, and `take` name (the caller has counted them:
// kCandidates at most), into its list of candidates; the list's last writes are seen after the next
// cluster barrier.
template <typename Look, typename Take>
__device__ void gather(Shared& s, const float* data, int count, uint32_t base, Look look, Take take) {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for_each_four(data, count, [&](const float(&v)[4], int i) {
        bool taken[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) taken[e] = look(v[e]) && v[e] != -INFINITY;
        if (taken[0] || taken[1] || taken[2] || taken[3])
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t rank = rank_of(key_of(v[e]), base + i + e);
                if (taken[e] && take(v[e], rank)) {
                    const uint32_t at = atomicAdd(&s.count, 1u);
                    if (at < kCandidates) s.mine[at] = rank;
                }
            }
    });
}

// The candidates of all CTAs and their weights, in this one's memory.
template <bool kWeighted>
__device__ int collect(cg::cluster_group& cluster, Shared& s, const Row& row) {
    const int ctas = cluster.num_blocks();
    int starts[kMaxCluster + 1];
    for_each_cta([&](int r) { starts[r + 1] = (int)cluster.map_shared_rank(&s, r < ctas ? r : 0)->count; });
    starts[0] = 0;
    for_each_cta([&](int r) { starts[r + 1] = starts[r] + (r < ctas ? starts[r + 1] : 0); });
    const int candidates = starts[kMaxCluster];
    for (int i = threadIdx.x; i < candidates; i += kThreads) {
        int from = 0, start = 0;
        for_each_cta([&](int r) {
            if (i >= starts[r] && i < starts[r + 1]) from = r, start = starts[r];
        });
        const uint64_t rank = cluster.map_shared_rank(&s, from)->mine[i - start];
        s.all[i] = rank;
        s.weight[i] = kWeighted ? weight_of(row, value_of((uint32_t)(rank >> 32))) : 1;
    }
    __syncthreads();
    return candidates;
}

// How many neighbouring threads share a candidate: a power of two, so that all have one if there are enough.
__device__ __forceinline__ int lanes_of(int candidates, int threads) {
    int lanes = 1;
    while (lanes < 32 && 2 * lanes * candidates <= threads) lanes *= 2;
    return lanes;
}

// A threshold search whose first step left too many elements: the rank of the last one that is kept.
template <bool kWeighted>
__device__ uint64_t search(cg::cluster_group& cluster, Shared& s, const float* data, int count, uint32_t base, const Row& row,
                           uint64_t floor, uint64_t need, Found found, int& buffer) {
    uint64_t above = found.before;  // mass of the ranks above `high`
    uint64_t low = floor, high = ~0ull;
    if (found.inside <= kCandidates) {
        gather(s, data, count, base, [&](float v) { return first_bin(row, v) == found.bin; },
               [&](float v, uint64_t rank) { return rank >= floor && counted<kWeighted>(row, v); });
    } else {
        if (threadIdx.x == 0) {
            s.low = ~0ull;
            s.high = 0;
        }
        __syncthreads();
        uint64_t my_low = ~0ull, my_high = 0;
        for_each(data, count, [&](float v, int i) {
            const uint64_t rank = rank_of(key_of(v), base + i);
            if (rank < floor || first_bin(row, v) != found.bin || (kWeighted && weight_of(row, v) == 0)) return;
            my_low = my_low < rank ? my_low : rank;
            my_high = my_high > rank ? my_high : rank;
        });
        atomicMin((unsigned long long*)&s.low, (unsigned long long)my_low);
        atomicMax((unsigned long long*)&s.high, (unsigned long long)my_high);
        cluster.sync();
        low = ~0ull;
        high = 0;
        for (int r = 0; r < (int)cluster.num_blocks(); ++r) {  // seldom: many equal logits
            const Shared* other = cluster.map_shared_rank(&s, r);
            low = low < other->low ? low : other->low;
            high = high > other->high ? high : other->high;
        }
        // bins of the rank inside [low, high]; a bin of a range below 512 holds one element
        while (true) {
            int shift = 0;
            while ((high - low) >> shift >= kBins) ++shift;
            clear_bins(s);
            uint32_t(*hist)[kBins] = s.hist;
            for_each(data, count, [&](float v, int i) {
                const uint64_t rank = rank_of(key_of(v), base + i);
                if (rank < low || rank > high) return;
                const uint64_t w = kWeighted ? weight_of(row, v) : 1;
                if (w == 0) return;
                const uint32_t bin = (uint32_t)((high - rank) >> shift);
                atomicAdd(&hist[0][bin], 1u);
                if (kWeighted) add_weight(hist, bin, w);
            });
            uint64_t rest = need - above;
            const Found next = scan_bins<kWeighted>(cluster, s, buffer, rest, 0.0f);
            above += next.before;
            high -= (uint64_t)next.bin << shift;
            const uint64_t width = ((uint64_t)1 << shift) - 1;
            low = high - low > width ? high - width : low;
            if (next.inside <= kCandidates) break;
        }
        // `low` is the rank of an element with weight: all above have some
        gather(s, data, count, base, [&](float v) { return first_bin(row, v) == found.bin; },
               [&](float, uint64_t rank) { return rank >= low && rank <= high; });
    }
    cluster.sync();
    const int candidates = collect<kWeighted>(cluster, s, row);
    // the element with which the running mass reaches `need`: the candidates are shared by all threads of the cluster
    const int ctas = cluster.num_blocks(), threads = ctas * kThreads, me = cluster.block_rank() * kThreads + threadIdx.x;
    const int lanes = lanes_of(candidates, threads), lane = me & (lanes - 1);
    for (int base = 0; base < candidates; base += threads / lanes) {
        const int i = base + me / lanes;
        const uint64_t rank = i < candidates ? s.all[i] : 0;
        uint64_t sum = 0;
        for (int j = lane; j < candidates; j += lanes) sum += s.all[j] > rank ? s.weight[j] : 0;
        for (int d = lanes >> 1; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        const uint64_t before = above + sum;
        if (i < candidates && lane == 0 && before < need && before + s.weight[i] >= need)
            for (int r = 0; r < ctas; ++r) cluster.map_shared_rank(&s, r)->found = rank;
    }
    cluster.sync();  // found is written, and nobody still reads this CTA's candidates
    const uint64_t rank = s.found;
    __syncthreads();
    return rank;
}

__device__ __forceinline__ uint64_t border_of(float u, uint64_t total) {
    // a sum exceeds u * total exactly if it exceeds the largest integer that is not above it
    return u >= 1.0f ? total - 1 : u > 0.0f ? share_of(u, total, false) : 0;
}

__device__ __forceinline__ float logprob_of(const Row& row, float v, uint64_t total) {
    return (float)(exponent_of(row, v) - log((double)total / kOne));
}

// The rest of a row whose candidates are few, in one CTA: ranked, cut by top-k, top-p (of row_total,
// or, where that is 0, of what top-k keeps) and min-p, and summed in vocabulary order.  Quadratic in
// the number of candidates, each for one to 32 neighbouring threads.
__device__ void finish_few(cg::cluster_group& cluster, Shared& s, const Params& p, const Row& row, int row_index, int top_k,
                           float top_p, double least, uint64_t row_total) {
    const int t = threadIdx.x, warp = t >> 5;
    const int candidates = collect<true>(cluster, s, row);
    const int lanes = lanes_of(candidates, kThreads), lane = t & (lanes - 1), i = t / lanes;
    const bool present = i < candidates;
    const uint64_t rank = present ? s.all[i] : 0;
    uint64_t weight = present ? s.weight[i] : 0;
    auto group_sum = [&](auto v) {
        for (int d = lanes >> 1; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        return v;
    };
    auto total_of_kept = [&]() {
        uint64_t sum = warp_total(lane == 0 ? weight : 0);
        __syncthreads();
        if ((t & 31) == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s.warp_sum[w];
        return sum;
    };
    int place = 0;
    uint64_t before = 0;
    if (present)
        for (int j = lane; j < candidates; j += lanes)
            if (s.all[j] > rank) {
                ++place;
                before += s.weight[j];
            }
    place = group_sum(place);
    before = group_sum(before);
    if (top_k > 0 && place >= top_k) weight = 0;
    if (top_p < 1.0f) {
        const uint64_t total = row_total ? row_total : total_of_kept();
        if (before >= (top_p > 0.0f ? share_of(top_p, total, true) : 1)) weight = 0;
    }
    const float value = value_of((uint32_t)(rank >> 32));
    if ((double)weight < least && value != row.top) weight = 0;
    const uint64_t total = total_of_kept();  // between its barriers everyone has read s.weight
    const uint64_t border = border_of(p.uniforms[row_index], total);
    if (present && lane == 0) s.weight[i] = weight;
    __syncthreads();
    uint64_t running = 0;
    if (weight != 0)  // the same for all threads of a candidate
        for (int j = lane; j < candidates; j += lanes)
            if ((uint32_t)s.all[j] > (uint32_t)rank) running += s.weight[j];  // a lower index has the larger complement
    running = group_sum(running);
    if (weight != 0 && lane == 0 && running <= border && running + weight > border) {
        p.tokens[row_index] = (long long)(0xFFFFFFFFu - (uint32_t)rank);
        p.logprobs[row_index] = logprob_of(row, value, total);
    }
}

// A row's slice into shared memory as fp32, filled up to whole quadruples with minus infinity; returns
// the largest of the thread's elements, or NaN if one of them is.
__device__ float load_slice(const Params& p, int64_t at, int count, float* data) {
    const int t = threadIdx.x;
    float top = -INFINITY;
    const int step = p.bf16 ? 8 : 4, whole = p.vector ? count / step * step : 0;
    if (p.bf16) {
        const __nv_bfloat16* source = reinterpret_cast<const __nv_bfloat16*>(p.logits) + at;
#pragma unroll 4
        for (int i = 8 * t; i < whole; i += 8 * kThreads) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(source + i));
            const float4 lo = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u),
                                          __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
            const float4 hi = make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xFFFF0000u),
                                          __uint_as_float(u.w << 16), __uint_as_float(u.w & 0xFFFF0000u));
            reinterpret_cast<float4*>(data + i)[0] = lo;
            reinterpret_cast<float4*>(data + i)[1] = hi;
            top = max_nan(top, max_nan(max_nan(lo.x, lo.y), max_nan(lo.z, lo.w)));
            top = max_nan(top, max_nan(max_nan(hi.x, hi.y), max_nan(hi.z, hi.w)));
        }
#pragma unroll 4
        for (int i = whole + t; i < count; i += kThreads) top = max_nan(top, data[i] = __bfloat162float(source[i]));
    } else {
        const float* source = reinterpret_cast<const float*>(p.logits) + at;
#pragma unroll 4
        for (int i = 4 * t; i < whole; i += 4 * kThreads) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(source + i));
            *reinterpret_cast<float4*>(data + i) = v;
            top = max_nan(top, max_nan(max_nan(v.x, v.y), max_nan(v.z, v.w)));
        }
#pragma unroll 4
        for (int i = whole + t; i < count; i += kThreads) top = max_nan(top, data[i] = source[i]);
    }
    if (t < 4 && count + t < (count + 3) / 4 * 4) data[count + t] = -INFINITY;
    return top;
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& s = *reinterpret_cast<Shared*>(raw);
    float* data = reinterpret_cast<float*>(raw + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = cluster.num_blocks(), rank_in_cluster = cluster.block_rank();
    const int row_index = blockIdx.x / ctas;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int first = min(rank_in_cluster * p.slice, p.vocabulary);
    const int count = min(p.slice, p.vocabulary - first);
    float top = load_slice(p, (int64_t)row_index * p.ld + first, count, data);
    if (t == 0) s.first_top = 0xFFFFFFFFu;
    if (t < 8) s.power[t] = exp2(0.125 * t);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (lane == 0) s.warp_top[warp] = top;
    __syncthreads();
    if (warp == 0) {
        top = s.warp_top[lane % kWarps];
#pragma unroll
        for (int d = 8; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        if (lane == 0) s.cta_top = top;
    }
    cluster.sync();
    float tops[kMaxCluster];
    for_each_cta([&](int r) { tops[r] = cluster.map_shared_rank(&s, r < ctas ? r : 0)->cta_top; });
    top = tops[0];
    for_each_cta([&](int r) { top = max_nan(top, tops[r]); });
    Row row;
    row.power = s.power;
    row.top = top;
    const float temperature = p.temperature_dev ? p.temperature_dev[row_index] : p.temperature;
    const int top_k = p.top_k_dev ? p.top_k_dev[row_index] : p.top_k;
    const float top_p = p.top_p_dev ? p.top_p_dev[row_index] : p.top_p;
    const float min_p = fmaxf(p.min_p_dev ? p.min_p_dev[row_index] : p.min_p, 0.0f);  // a NaN cuts nothing, everywhere
    if (top != top || top == -INFINITY) {
        if (rank_in_cluster == 0 && t == 0) {
            p.tokens[row_index] = -1;
            p.logprobs[row_index] = __uint_as_float(0x7FC00000u);
        }
        cluster.sync();  // nobody leaves while its maximum may still be read
        return;
    }
    if (!(temperature > 0.0f) || top_k == 1) {
        // the first of the largest logits
        for_each(data, count, [&](float v, int i) {
            if (v == top) atomicMin(&s.first_top, (uint32_t)(first + i));
        });
        cluster.sync();
        if (rank_in_cluster == 0 && t == 0) {
            uint32_t index = 0xFFFFFFFFu;
            for (int r = 0; r < ctas; ++r) index = min(index, cluster.map_shared_rank(&s, r)->first_top);
            p.tokens[row_index] = index;
            p.logprobs[row_index] = 0.0f;
        }
        cluster.sync();
        return;
    }
    row.inverse = 1.0 / (double)temperature;
    row.bin_scale = fminf(kBinsPerUnit / temperature, 1e30f);

    const double least = (double)min_p * kOne;
    uint64_t threshold = 0;
    int buffer = 0;
    bool few = false, in_bins = false;
    uint64_t row_total = 0;
    Found found;
    if (top_k > 0 && top_k < p.vocabulary) {
        uint64_t need = top_k;
        found = first_step<false>(cluster, s, data, count, first, row, 0, need, 0.0f, buffer);
        if (found.total > need) {
            few = found.through <= kFew;
            if (!few) threshold = search<false>(cluster, s, data, count, first, row, 0, need, found, buffer);
        }
    }
    if (!few && top_p < 1.0f) {
        uint64_t need = 1;
        found = first_step<true>(cluster, s, data, count, first, row, threshold, need, top_p, buffer);
        few = threshold == 0 && found.through <= kFew;
        if (few)
            row_total = found.total;
        else {
            in_bins = found.inside <= kCandidates;  // the search adds no histogram to the first step's
            threshold = search<true>(cluster, s, data, count, first, row, threshold, need, found, buffer);
        }
    }
    if (few) {
        gather(s, data, count, first, [&](float v) { return first_bin(row, v) <= found.bin; },
               [&](float v, uint64_t) { return row_total == 0 || counted<true>(row, v); });
        cluster.sync();
        if (rank_in_cluster == 0)
            finish_few(cluster, s, p, row, row_index, row_total ? 0 : top_k, top_p, least, row_total);
        cluster.sync();  // nobody leaves while its candidates may still be read
        return;
    }

    // Every thread has neighbouring elements, at most 64, and takes them in an order of its own, so that a
    // warp's reads meet few banks twice.  Which are kept is known before any weight is computed: in a
    // nucleus, few.
    const int own = max((count + kThreads - 1) / kThreads, 1), from = min(t * own, count), to = min(from + own, count);
    auto kept = [&](float v, int i) {
        return v != -INFINITY && rank_of(key_of(v), (uint32_t)(first + i)) >= threshold;
    };
    auto kept_weight = [&](float v) -> uint64_t {
        const uint64_t w = weight_of(row, v);
        return v == row.top || (double)w >= least ? w : 0;
    };
    auto sum_own = [&]() {
        uint64_t mask = 0, sum = 0;
        for (int e = 0, at = lane % own; e < own; ++e, at = at + 1 < own ? at + 1 : 0) {
            const int i = from + at;
            if (i < to && kept(data[i], i)) mask |= (uint64_t)1 << at;
        }
        while (mask) {
            const int at = __ffsll((long long)mask) - 1;
            mask &= mask - 1;
            sum += kept_weight(data[from + at]);
        }
        return sum;
    };
    // What this CTA keeps: the bins above the one with top-p's threshold and, of that one, the
    // candidates down to it; where there is no such step, or min-p cuts too, the sum over its slice.
    const bool from_bins = in_bins && !(least > 0.0);
    uint64_t sum = 0;
    if (from_bins) {
        if (t < (int)found.bin) sum = s.bin_weight[buffer ^ 1][t];
        for (int i = t; i < (int)s.count; i += kThreads)
            if (s.mine[i] >= threshold) sum += weight_of(row, value_of((uint32_t)(s.mine[i] >> 32)));
    } else {
        sum = sum_own();
    }
    const uint64_t warp_sum = warp_total(sum);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = warp_sum;
    __syncthreads();
    if (t == 0) {
        uint64_t all = 0;
        for (int w = 0; w < kWarps; ++w) all += s.warp_sum[w];
        s.cta_sum = all;
    }
    cluster.sync();
    uint64_t sums[kMaxCluster], total = 0, before = 0;
    for_each_cta([&](int r) { sums[r] = cluster.map_shared_rank(&s, r < ctas ? r : 0)->cta_sum; });
    for_each_cta([&](int r) {
        if (r < ctas) total += sums[r];
        if (r < rank_in_cluster) before += sums[r];
    });
    const uint64_t border = border_of(p.uniforms[row_index], total);
    if (before <= border && before + s.cta_sum > border) {  // the token is in this CTA's slice
        if (from_bins) {
            sum = sum_own();
            const uint64_t sum_of_warp = warp_total(sum);
            __syncthreads();
            if (lane == 0) s.warp_sum[warp] = sum_of_warp;
            __syncthreads();
        }
        for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
        if (before <= border && before + s.warp_sum[warp] > border) {  // ... in this warp's elements
            const uint64_t running = before + warp_running(sum);
            const uint32_t owner = __ballot_sync(0xFFFFFFFFu, running - sum <= border && running > border);
            const int start = __shfl_sync(0xFFFFFFFFu, from, __ffs(owner) - 1), stop = __shfl_sync(0xFFFFFFFFu, to, __ffs(owner) - 1);
            before = __shfl_sync(0xFFFFFFFFu, running - sum, __ffs(owner) - 1);
            for (int i0 = start; i0 < stop; i0 += 32) {
                const int i = i0 + lane;
                const uint64_t w = i < stop && kept(data[i], i) ? kept_weight(data[i]) : 0;
                const uint64_t through = before + warp_running(w);
                if (w != 0 && through > border && through - w <= border) {
                    p.tokens[row_index] = first + i;
                    p.logprobs[row_index] = logprob_of(row, data[i], total);
                }
                before = __shfl_sync(0xFFFFFFFFu, through, 31);
            }
        }
    }
    cluster.sync();  // nobody leaves while its sums may still be read
}

int launch(Params p, int64_t rows, cudaStream_t stream) {
    int ctas = 1;
    while (ctas < kMaxCluster && p.vocabulary > 4096 * ctas) ctas *= 2;
    p.slice = (int)(((p.vocabulary + ctas - 1) / ctas + 7) / 8 * 8);
    const size_t bytes = sizeof(Shared) + (size_t)p.slice * sizeof(float);
    cudaError_t error = allow_shared<sample_kernel>((int)(sizeof(Shared) + kMaxVocabulary / kMaxCluster * sizeof(float)));
    if (error != cudaSuccess) return record_cuda_error(error);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = ctas;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    error = cudaLaunchKernelEx(&config, sample_kernel, p);
    if (error != cudaSuccess) return record_cuda_error(error);
    return check_launch();
}

}  // namespace sample
}  // namespace ue5m3

extern "C" int ue5m3_sample_tokens(const void* logits, int dtype, int64_t rows, int64_t vocabulary, int64_t ld,
                                   const float* uniforms, const float* temperature_dev, float temperature,
                                   const int* top_k_dev, int top_k, const float* top_p_dev, float top_p,
                                   const float* min_p_dev, float min_p, int64_t* tokens, float* logprobs,
                                   void* stream) {
    using namespace ue5m3;
    if (!logits || !uniforms || !tokens || !logprobs || rows <= 0 || vocabulary <= 0 || ld < vocabulary ||
        (dtype != UE5M3_DTYPE_BF16 && dtype != UE5M3_DTYPE_FP32))
        return UE5M3_ERR_INVALID_ARGUMENT;
    if (vocabulary > sample::kMaxVocabulary || rows > (1 << 24)) {
        record_error_text("at most 2^18 logits per row and 2^24 rows");
        return UE5M3_ERR_TOO_LARGE;
    }
    const int element = dtype == UE5M3_DTYPE_FP32 ? 4 : 2;
    if ((uintptr_t)logits % element) return UE5M3_ERR_ALIGNMENT;
    sample::Params p;
    p.logits = logits;
    p.ld = ld;
    p.uniforms = uniforms;
    p.temperature_dev = temperature_dev;
    p.top_k_dev = top_k_dev;
    p.top_p_dev = top_p_dev;
    p.min_p_dev = min_p_dev;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.tokens = (long long*)tokens;
    p.logprobs = logprobs;
    p.vocabulary = (int)vocabulary;
    p.bf16 = dtype == UE5M3_DTYPE_BF16;
    p.vector = (uintptr_t)logits % 16 == 0 && (ld * element) % 16 == 0;
    return sample::launch(p, rows, (cudaStream_t)stream);
}
