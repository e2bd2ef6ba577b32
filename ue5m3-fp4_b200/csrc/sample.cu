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
// What bounds it: a batch of rows, reading the logits and one fp64 exponential per logit that a sum
// needs; a single row, the latency of about ten steps.  A cluster of up to eight CTAs holds a row in
// shared memory, so that it is read from memory once however many steps follow.  A step of a
// threshold search is a histogram of 512 bins over the row, summed over the cluster through
// distributed shared memory by every CTA for itself (one cluster barrier per step).  The first
// step's bins are linear in (max - l) / T, which spreads real logits (bins of the integer order
// would put a fifth of a row into one of them); the elements of the bin that holds the threshold
// are then few enough to be ranked against one another, or the search goes on inside it with bins
// of the 64-bit rank (many equal logits).
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
    uint32_t hist[2][4][kBins];  // [buffer][count, weight bits 0..14, 15..29, 30..44]
    uint64_t mine[kCandidates];  // this CTA's candidates
    uint64_t all[kCandidates];
    uint64_t weight[kCandidates];
    uint64_t warp_sum[kWarps];
    uint64_t cta_sum;
    uint64_t found, found_before;
    uint64_t low, high;          // bounds of the ranks in a bin (this CTA's)
    uint32_t top_key, top_index, bad, count;
    uint32_t found_bin, found_count;
};

// logits in integer order: a larger logit has a larger key
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint64_t rank_of(uint32_t key, uint32_t index) {
    return (uint64_t)key << 32 | (0xFFFFFFFFu - index);
}

// 2^44 exp(z), z <= 0, to the nearest integer: Taylor's polynomial of degree 11 on
// |r| <= ln(2) / 2, whose remainder is below 2^-47 of the value.
__device__ __forceinline__ uint64_t weight_of(double z) {
    if (!(z > -31.2)) return 0;  // below half a unit
    const double n = rint(z * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, z);  // |n| <= 45: the constant's rounding costs 2^-49
    double e = 1.0 / 39916800.0;
    e = fma(e, r, 1.0 / 3628800.0);
    e = fma(e, r, 1.0 / 362880.0);
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const double scaled = __hiloint2double(__double2hiint(e) + (((int)n + 44) << 20), __double2loint(e));
    return (uint64_t)__double2ull_rn(scaled);
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
    float top;         // the largest logit
    double inverse;    // 1 / T
    float bin_scale;   // kBinsPerUnit / T, finite
};

__device__ __forceinline__ double exponent_of(const Row& row, float v) {
    if (v == row.top) return 0.0;  // also where both are infinite
    return ((double)v - (double)row.top) * row.inverse;
}

__device__ __forceinline__ uint64_t weight_of(const Row& row, float v) {
    if (v == -INFINITY) return 0;
    return weight_of(exponent_of(row, v));
}

__device__ __forceinline__ uint32_t first_bin(const Row& row, float v) {
    if (v == row.top) return 0;
    const float bin = (row.top - v) * row.bin_scale;  // monotone in v: each step rounds monotonely
    return bin < (float)(kBins - 1) ? (uint32_t)bin : kBins - 1;
}

// A threshold search over the elements with rank >= floor: by number (kWeighted false, the
// need-th largest) or by weight (the first one, in descending order, with which the running weight
// reaches `need`; for top-p, need is a share of the weight of all of them).  Every CTA of the
// cluster runs it with the same arguments and gets the same answer.  0 = everything is kept.
template <bool kWeighted>
__device__ uint64_t find_threshold(cg::cluster_group& cluster, Shared& s, const float* data, int count, uint32_t base,
                                   const Row& row, uint64_t floor, uint64_t need, float share, int& buffer) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int ctas = cluster.num_blocks();
    uint64_t low = floor, high = ~0ull;  // ranks under consideration
    uint64_t above = 0;                  // mass of the ranks above `high`
    int shift = 0;
    uint32_t bin1 = 0;
    for (int level = 0;; ++level) {
        uint32_t(*hist)[kBins] = s.hist[buffer];
        for (int i = 0; i < 4; ++i) hist[i][t] = 0;
        __syncthreads();
        for (int i = t; i < count; i += kThreads) {
            const float v = data[i];
            if (v == -INFINITY) continue;
            const uint64_t rank = rank_of(key_of(v), base + i);
            if (rank < low || rank > high) continue;
            const uint32_t bin = level == 0 ? first_bin(row, v) : (uint32_t)((high - rank) >> shift);
            uint64_t w = 1;
            if (kWeighted) {
                w = weight_of(row, v);
                if (w == 0) continue;
                atomicAdd(&hist[1][bin], (uint32_t)(w & 0x7FFF));
                atomicAdd(&hist[2][bin], (uint32_t)(w >> 15 & 0x7FFF));
                atomicAdd(&hist[3][bin], (uint32_t)(w >> 30));
            }
            atomicAdd(&hist[0][bin], 1u);
        }
        cluster.sync();
        // every CTA sums the bins of all; thread = bin
        uint64_t mass = 0;
        uint32_t number = 0;
        for (int r = 0; r < ctas; ++r) {
            const Shared* other = cluster.map_shared_rank(&s, r);
            const uint32_t n = other->hist[buffer][0][t];
            number += n;
            if (kWeighted)
                mass += (uint64_t)other->hist[buffer][1][t] + ((uint64_t)other->hist[buffer][2][t] << 15) +
                        ((uint64_t)other->hist[buffer][3][t] << 30);
            else
                mass += n;
        }
        buffer ^= 1;
        uint64_t running = mass;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t from = __shfl_up_sync(0xFFFFFFFFu, running, d);
            if (lane >= d) running += from;
        }
        if (lane == 31) s.warp_sum[warp] = running;
        if (t == 0) s.found_bin = kBins;
        __syncthreads();
        uint64_t before = above, total = above;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s.warp_sum[w];
            total += s.warp_sum[w];
        }
        running += before;
        if (level == 0 && kWeighted) {
            // the running weight before the last kept element is below share * total
            need = share > 0.0f ? share_of(share, total, true) : 1;
        }
        if (total <= need && level == 0 && !kWeighted) {
            __syncthreads();
            return floor;  // no more than `need` elements
        }
        if (running >= need && running - mass < need) {
            s.found_bin = t;
            s.found_before = running - mass;
            s.found_count = number;
        }
        __syncthreads();
        const uint32_t bin = s.found_bin, inside = s.found_count;
        above = s.found_before;
        __syncthreads();
        if (level == 0)
            bin1 = bin;
        else {
            high -= (uint64_t)bin << shift;
            const uint64_t width = ((uint64_t)1 << shift) - 1;
            low = high - low > width ? high - width : low;
        }
        // the elements of the bin: ranked against one another when they are few
        const bool few = inside <= kCandidates;
        if (t == 0) {
            s.count = 0;
            s.low = ~0ull;
            s.high = 0;
        }
        __syncthreads();
        if (few || level == 0) {
            uint64_t my_low = ~0ull, my_high = 0;
            for (int i = t; i < count; i += kThreads) {
                const float v = data[i];
                if (v == -INFINITY) continue;
                const uint64_t rank = rank_of(key_of(v), base + i);
                if (rank < low || rank > high || (level == 0 && first_bin(row, v) != bin1)) continue;
                if (kWeighted && weight_of(row, v) == 0) continue;
                if (few)
                    s.mine[atomicAdd(&s.count, 1u)] = rank;
                else {
                    my_low = my_low < rank ? my_low : rank;
                    my_high = my_high > rank ? my_high : rank;
                }
            }
            if (!few) {
                atomicMin((unsigned long long*)&s.low, (unsigned long long)my_low);
                atomicMax((unsigned long long*)&s.high, (unsigned long long)my_high);
            }
        }
        if (few) break;
        if (level == 0) {
            cluster.sync();
            low = ~0ull;
            high = 0;
            for (int r = 0; r < ctas; ++r) {
                const Shared* other = cluster.map_shared_rank(&s, r);
                low = low < other->low ? low : other->low;
                high = high > other->high ? high : other->high;
            }
            cluster.sync();  // the bounds are rewritten by a later search
        }
        const uint64_t range = high - low;
        shift = 0;
        while (range >> shift >= kBins) ++shift;
    }
    cluster.sync();
    int candidates = 0;
    for (int r = 0; r < ctas; ++r) {
        const Shared* other = cluster.map_shared_rank(&s, r);
        const int n = (int)other->count;
        for (int i = t; i < n; i += kThreads) s.all[candidates + i] = other->mine[i];
        candidates += n;
    }
    __syncthreads();
    for (int i = t; i < candidates; i += kThreads)
        s.weight[i] = kWeighted ? weight_of(row, value_of((uint32_t)(s.all[i] >> 32))) : 1;
    __syncthreads();
    for (int i = t; i < candidates; i += kThreads) {
        const uint64_t rank = s.all[i];
        uint64_t before = above;
        for (int j = 0; j < candidates; ++j)
            if (s.all[j] > rank) before += s.weight[j];
        if (before < need && before + s.weight[i] >= need) s.found = rank;
    }
    cluster.sync();  // found, and nobody still reads this CTA's candidates
    const uint64_t found = s.found;
    __syncthreads();
    return found;
}

__device__ void load_slice(const Params& p, int64_t at, int count, float* data) {
    const int t = threadIdx.x;
    if (p.bf16) {
        const __nv_bfloat16* source = reinterpret_cast<const __nv_bfloat16*>(p.logits) + at;
        int i = 0;
        if (p.vector) {
            const uint4* wide = reinterpret_cast<const uint4*>(source);
            for (i = t; i < count / 8; i += kThreads) {
                const uint4 u = __ldg(wide + i);
                float4* to = reinterpret_cast<float4*>(data + 8 * i);
                to[0] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u),
                                    __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
                to[1] = make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xFFFF0000u),
                                    __uint_as_float(u.w << 16), __uint_as_float(u.w & 0xFFFF0000u));
            }
            for (i = count / 8 * 8 + t; i < count; i += kThreads) data[i] = __bfloat162float(source[i]);
        } else {
            for (i = t; i < count; i += kThreads) data[i] = __bfloat162float(source[i]);
        }
    } else {
        const float* source = reinterpret_cast<const float*>(p.logits) + at;
        if (p.vector) {
            const float4* wide = reinterpret_cast<const float4*>(source);
            for (int i = t; i < count / 4; i += kThreads) reinterpret_cast<float4*>(data)[i] = __ldg(wide + i);
            for (int i = count / 4 * 4 + t; i < count; i += kThreads) data[i] = source[i];
        } else {
            for (int i = t; i < count; i += kThreads) data[i] = source[i];
        }
    }
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& s = *reinterpret_cast<Shared*>(raw);
    float* data = reinterpret_cast<float*>(raw + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = cluster.num_blocks(), rank_in_cluster = cluster.block_rank();
    const int row_index = blockIdx.x / ctas;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int first = min(rank_in_cluster * p.slice, p.vocabulary);
    const int count = min(p.slice, p.vocabulary - first);
    load_slice(p, (int64_t)row_index * p.ld + first, count, data);
    if (t == 0) {
        s.top_key = 0;
        s.top_index = 0xFFFFFFFFu;
        s.bad = 0;
    }
    __syncthreads();

    // the largest logit, the lowest index that has it, and whether a NaN is among them
    uint64_t best = 0;
    bool bad = false;
    for (int i = t; i < count; i += kThreads) {
        const float v = data[i];
        bad |= v != v;
        const uint64_t rank = rank_of(key_of(v), (uint32_t)(first + i));
        best = best > rank ? best : rank;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, best, d);
        best = best > other ? best : other;
    }
    if (bad) s.bad = 1;
    if (lane == 0) s.warp_sum[warp] = best;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kWarps; ++w) best = best > s.warp_sum[w] ? best : s.warp_sum[w];
        s.cta_sum = best;
    }
    cluster.sync();
    best = 0;
    uint32_t any_bad = 0;
    for (int r = 0; r < ctas; ++r) {
        const Shared* other = cluster.map_shared_rank(&s, r);
        best = best > other->cta_sum ? best : other->cta_sum;
        any_bad |= other->bad;
    }
    cluster.sync();  // cta_sum and warp_sum are used again
    Row row;
    row.top = value_of((uint32_t)(best >> 32));
    const float temperature = p.temperature_dev ? p.temperature_dev[row_index] : p.temperature;
    const int top_k = p.top_k_dev ? p.top_k_dev[row_index] : p.top_k;
    const float top_p = p.top_p_dev ? p.top_p_dev[row_index] : p.top_p;
    const float min_p = p.min_p_dev ? p.min_p_dev[row_index] : p.min_p;
    if (any_bad || row.top == -INFINITY) {
        if (rank_in_cluster == 0 && t == 0) {
            p.tokens[row_index] = -1;
            p.logprobs[row_index] = __uint_as_float(0x7FC00000u);
        }
        return;
    }
    if (!(temperature > 0.0f) || top_k == 1) {
        if (rank_in_cluster == 0 && t == 0) {
            p.tokens[row_index] = (long long)(0xFFFFFFFFu - (uint32_t)best);
            p.logprobs[row_index] = 0.0f;
        }
        return;
    }
    row.inverse = 1.0 / (double)temperature;
    row.bin_scale = fminf(kBinsPerUnit / temperature, 1e30f);

    uint64_t threshold = 0;
    int buffer = 0;
    if (top_k > 0 && top_k < p.vocabulary)
        threshold = find_threshold<false>(cluster, s, data, count, first, row, threshold, (uint64_t)top_k, 0.0f, buffer);
    if (top_p < 1.0f)
        threshold = find_threshold<true>(cluster, s, data, count, first, row, threshold, 0, top_p, buffer);

    // the kept weight of every warp's run of the slice
    const double least = (double)min_p * kOne;
    auto kept_weight = [&](int i) -> uint64_t {
        const float v = data[i];
        if (rank_of(key_of(v), (uint32_t)(first + i)) < threshold) return 0;
        const uint64_t w = weight_of(row, v);
        return v != row.top && (double)w < least ? 0 : w;
    };
    const int run = (count + kThreads - 1) / kThreads * 32;
    const int from = min(warp * run, count), to = min(from + run, count);
    uint64_t sum = 0;
    for (int i = from + lane; i < to; i += 32) sum += kept_weight(i);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) s.warp_sum[warp] = sum;
    __syncthreads();
    if (t == 0) {
        uint64_t all = 0;
        for (int w = 0; w < kWarps; ++w) all += s.warp_sum[w];
        s.cta_sum = all;
    }
    cluster.sync();
    uint64_t total = 0, before = 0;
    for (int r = 0; r < ctas; ++r) {
        const uint64_t of = cluster.map_shared_rank(&s, r)->cta_sum;
        if (r < rank_in_cluster) before += of;
        total += of;
    }
    // a sum exceeds u * total exactly if it exceeds the largest integer that is not above it
    const float u = p.uniforms[row_index];
    const uint64_t border = u >= 1.0f ? total - 1 : u > 0.0f ? share_of(u, total, false) : 0;
    for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
    if (before <= border && before + s.warp_sum[warp] > border) {
        // this warp's run holds the token
        for (int i0 = from; i0 < to; i0 += 32) {
            const int i = i0 + lane;
            const uint64_t w = i < to ? kept_weight(i) : 0;
            uint64_t running = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t other = __shfl_up_sync(0xFFFFFFFFu, running, d);
                if (lane >= d) running += other;
            }
            if (w != 0 && before + running > border && before + running - w <= border) {
                p.tokens[row_index] = first + i;
                p.logprobs[row_index] = (float)(exponent_of(row, data[i]) - log((double)total / kOne));
            }
            before += __shfl_sync(0xFFFFFFFFu, running, 31);
            if (before > border) break;
        }
    }
    cluster.sync();  // nobody leaves while its sums may still be read
}

int launch(Params p, int64_t rows, cudaStream_t stream) {
    int ctas = 1;
    while (ctas < kMaxCluster && p.vocabulary > 4096 * ctas) ctas *= 2;
    p.slice = (int)(((p.vocabulary + ctas - 1) / ctas + 7) / 8 * 8);
    const size_t bytes = sizeof(Shared) + (size_t)p.slice * sizeof(float);
    cudaError_t error = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(sizeof(Shared) + kMaxVocabulary / kMaxCluster * sizeof(float)));
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
