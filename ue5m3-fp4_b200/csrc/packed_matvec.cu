// A few rows of activations times a packed FP4 weight (the product of a decode step):
//   out[t, n] = dec * sum_k x[t, k] * p[n, k] * s[n, k / B]  (+ bias[n])
// with E2M1 payloads p and UE5M3 block scales s as the quantizer stores them (1 x B blocks or
// B x B tiles) and the activations as they are: no activation is quantized here.
//
// Arithmetic.  p * s has at most six significant bits and lies between 2^-18 and 2^19, so
// p * (s / 16) is EXACT in fp16 for every code and every scale byte.  x does not fit fp16 as it
// is: 128 consecutive elements of a row share a power of two that brings their largest one to
// [2^14, 2^15).  A bf16 element whose exponent is no more than 31 below that of the largest one is then
// exact in fp16, and an fp32 element down to 37 in three fp16 parts (11 bits each) with a product of
// its own each.  Tensor cores (mma.m16n8k16, weights as the 16-row operand, activations as the 8
// columns) sum 128 products in fp32; the power of two is multiplied back when that sum joins the fp32
// total.  The order of all sums is fixed by the sizes: the same call gives the same bits.
// Where a row's 128 elements span more than that (a wide column), they count as zeros there and enter in a
// second product of their own, after the others: as they are, in bf16 (fp32: three bf16 parts), with the same
// weights, which bf16 holds as exactly as fp16.  (Every chunk this way: 19 operations in place of 8 to
// decode eight codes.)  Of squared ReLUs of normal numbers one column in 360 is wide: 8 x 4096 x 21504 takes
// 23.8 us with them, 21.5 without; 64 x 4096 x 21504 62.7 and 53.9; with nothing but wide columns 42 and 259.
//
// What bounds it: reading the codes, 0.5 byte per weight element, plus the scales.  Decoding costs
// one cvt.rn.f16x2.e2m1x2 and one packed multiply per two weights.
//
// Up to eight tokens.  Every CTA owns N / gridDim rows (not a multiple of 16: missing rows of the last
// 16-row tile are not loaded, so that all SMs read the same number of bytes), every one of its
// warps w the 128-element chunks w, w + 16, ... of the reduction axis.  A warp keeps the activations
// of its chunks in registers (as mma fragments) while it walks over the CTA's rows; the sums of
// the 16 warps meet in shared memory once per block of rows.  Measured: 1 x 21504 x 4096: 15.5 us,
// 2.9 TB/s of 6.5 (fp32 22.3); 8 x 4096 x 21504: 20.6 us, 2.3 TB/s (fp32 36.3); 1 x 512 x 4096: 4.8 us.
// Of its active cycles the first one issues in 55 % of the slots and keeps the ALU, which decodes, busy
// for 41 %; launch, conversion of the activations (a look at their range costs 0.3 us of it) and
// the sums at the end do not overlap with the walk.  Rows that start anywhere come as aligned pieces
// and are shifted into place: 1 x 21504 x 4095: 29 us (word by word into registers 51, pieces per warp
// and chunk 34).
//
// More tokens.  There every CTA would convert all activations for its few rows: a short kernel writes
// them as fragments once (tokens x K x 2 bytes, three times that for fp32), and CTAs of 128 rows take
// them through a ring in shared memory, next to codes and scales, four warps of 32 rows for each of
// two halves of the chunks.  Measured: 64 x 18560 x 4096: 105 -> 41.1 us, 237 TFLOP/s, an mma in 17.8 active
// cycles of each quarter of an SM, the tensor pipe 46 % busy; 33 x 4096 x 4096: 31 -> 13.7; 60 x 2718 x 15245,
// whose rows start anywhere: 258 -> 47; fp32, three products each, 40 x 2000 x 3001: 47.5 -> 17.5,
// 64 x 4096 x 4096: 30.5; 2048 x 21504 x 4096, the weight decoded again for every 64 rows: 1444.  Bound by the
// products' issue from 32 tokens on, by decoding and the fragments' way from L2 below
// (16 x 21504 x 4096: 32.7 us).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "abi_common.cuh"

namespace ue5m3 {
namespace matvec {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kFewTokens = 8;          // up to here a CTA converts the activations itself
constexpr int kChunk = 128;          // reduction elements of one warp step: 64 bytes of a row's codes
constexpr int kPartialFloats = 20480;  // 80 KiB of partial sums per CTA
constexpr int kRing = 3;             // tiles of codes and scales in shared memory, 36 KiB each at two chunks per warp

// one chunk of eight tokens, 36 words for every 32 elements: the lanes' reads meet no bank twice
constexpr int kStageWords = 8 * 4 * 36;
constexpr int kStagePieces = kWarps * kStageWords / 4;

// 16-byte pieces of a ring slot: the codes of 16 rows and `depth` chunks per warp, and their scales
// (16 rows x 8 bytes, half of it used for blocks of 32)
__host__ __device__ constexpr int slot_pieces(int depth) { return depth * 2 * kThreads + kWarps * depth * 8; }
// ... and of one where rows start anywhere: for 16 rows the aligned pieces that hold their bytes of the 16
// warps' chunks, codes and scales
constexpr int kRowPieces = kWarps * kChunk / 2 / 16 + 1, kRowScalePieces = kWarps * kChunk / 16 / 16 + 1;
constexpr int kRowSlot = 16 * (kRowPieces + kRowScalePieces);

struct Params {
    const void* x;
    int64_t ldx;
    const uint8_t* codes;
    const uint8_t* scales;
    const void* bias;
    void* out;
    int64_t ldo;
    int64_t code_stride;   // bytes per row of codes
    int64_t scale_stride;  // bytes per row of scales
    int tokens, rows, k;
    int row_shift;         // log2 of the rows that share a scale row: 0, 4 or 5
    int split;             // CTAs of a cluster that share the reduction axis
    int rows_per_block;    // rows of one pass over shared memory, a multiple of 16
    int row_blocks;        // more than eight tokens: blocks of rows, each for one CTA or cluster
    int vector_x;          // rows of x start on 16-byte boundaries and hold whole vectors
    int bias_fp32, out_fp32;
    float factor;          // 16 * dec
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// eight codes -> four fp16 pairs, exactly
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t word, uint32_t (&d)[4]) {
    asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\ncvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\ncvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(word));
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// A scale byte E<<3|M as the fp16 pair (s/16, s/16): read as the top bits of an fp32 the byte is
// s * 2^-112, subnormal bytes included, and s/16 is exact in fp16 for all 256 bytes.
__device__ __forceinline__ uint32_t scale_half2(uint32_t byte) {
    const float v = __uint_as_float(byte << 20) * 0x1p108f;
    const __half2 h = __floats2half2_rn(v, v);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// What a lane brings of a chunk's activations, as they are in memory: 32 consecutive elements of one
// token, zero behind the end.
template <bool kFp32>
struct Raw {
    uint32_t words[kFp32 ? 32 : 16];
};

template <bool kFp32>
__device__ __forceinline__ Raw<kFp32> load_raw(const Params& p, int token, bool wanted, int chunk) {
    constexpr int kWords = kFp32 ? 32 : 16, kSize = kFp32 ? 4 : 2;
    const int k0 = chunk * kChunk + 32 * (threadIdx.x & 3);
    const bool present = wanted && k0 < p.k;
    const uint8_t* row = reinterpret_cast<const uint8_t*>(p.x) + (present ? (int64_t)token * p.ldx + k0 : 0) * kSize;
    Raw<kFp32> raw;
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw.words[i] = 0;
    if (!present) return raw;
    if (p.vector_x && k0 + 32 <= p.k) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i)
            *reinterpret_cast<uint4*>(raw.words + 4 * i) = __ldg(reinterpret_cast<const uint4*>(row) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const bool in = k0 + i < p.k;
            if constexpr (kFp32)
                raw.words[i] = in ? __ldg(reinterpret_cast<const uint32_t*>(row) + i) : 0;
            else
                raw.words[i / 2] |= (in ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + i) : 0u) << (16 * (i & 1));
        }
    }
    return raw;
}

// The same by a whole warp, for activations whose rows do not start on 16-byte boundaries, as those of
// an odd width: tokens token0 ... token0 + here - 1 (eight at most) side by side, 32 elements at a time,
// through `mine` (kStageWords of shared memory).
template <bool kFp32>
__device__ __forceinline__ Raw<kFp32> load_staged(const Params& p, int token0, int here, int chunk, uint32_t* mine) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < here)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = chunk * kChunk + q * 32 + lane;
                const int64_t at = (int64_t)(token0 + j) * p.ldx + k;
                uint32_t word = 0;
                if (k < p.k)
                    word = kFp32 ? __ldg(reinterpret_cast<const uint32_t*>(p.x) + at)
                                 : (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p.x) + at);
                mine[j * 144 + q * 36 + lane] = word;
            }
    __syncwarp();
    Raw<kFp32> raw;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint4 w = g < here ? *reinterpret_cast<const uint4*>(mine + g * 144 + c * 36 + 4 * i) : make_uint4(0, 0, 0, 0);
        if constexpr (kFp32) {
            raw.words[4 * i] = w.x, raw.words[4 * i + 1] = w.y, raw.words[4 * i + 2] = w.z, raw.words[4 * i + 3] = w.w;
        } else {
            raw.words[2 * i] = w.x | w.y << 16;
            raw.words[2 * i + 1] = w.z | w.w << 16;
        }
    }
    return raw;
}

// The largest magnitude among the 128 elements of a lane's token, and the smallest of this lane's that are
// not zero, less one unit: as the bits of an fp32.  Three operations for two bf16 elements, two for an fp32 one.
template <bool kFp32>
__device__ __forceinline__ void range_of(const Raw<kFp32>& raw, uint32_t& top, uint32_t& least) {
    least = 0xFFFFFFFFu;
    if constexpr (kFp32) {
        float most = 0.0f;  // a NaN does not count
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float a = fabsf(__uint_as_float(raw.words[i])), b = fabsf(__uint_as_float(raw.words[i + 1]));
            asm("max.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(a), "f"(b));
            // twice the magnitude: the sign leaves the word
            least = __vimin3_u32(least, 2 * raw.words[i] - 1, 2 * raw.words[i + 1] - 1);
        }
        top = __float_as_uint(most);
        least >>= 1;
    } else {
        uint32_t two = 0;  // a NaN's bits are larger than all numbers'
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint32_t a = raw.words[i] & 0x7FFF7FFFu, b = raw.words[i + 1] & 0x7FFF7FFFu;
            two = __vimax3_u16x2(two, a, b);
            least = __viaddmin_u16x2(a, 0xFFFFFFFFu, least);
            least = __viaddmin_u16x2(b, 0xFFFFFFFFu, least);
        }
        top = max(two << 16, two & 0xFFFF0000u);
        least = min(least << 16, least & 0xFFFF0000u);
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
}

// Whether one of the lane's elements does not fit next to its chunk's largest one: with exponents e and f it
// becomes a multiple of 2^(e - f + 7) (fp32: 2^(e - f - 9)), the last part holds multiples of 2^-24 (2^-46).  Beside
// an infinity or a NaN it does not matter.
template <bool kFp32>
__device__ __forceinline__ bool too_small(uint32_t top, uint32_t least) {
    constexpr uint32_t kSpan = (kFp32 ? 37 : 31) << 23, kUnit = kFp32 ? 1 : 1 << 16;
    const uint32_t exponent = top & 0x7F800000u;
    return exponent > kSpan && exponent < 0x7F800000u && least < exponent - kSpan - kUnit;
}

// One chunk's activations as mma B fragments (fp32: three, of 11 bits each, the second to be multiplied
// by 2^-11, the third by 2^-22), and the factor that undoes the chunk's power of two.  Lane (g, c) =
// (lane / 4, lane % 4) brings column g and elements 32 c ... 32 c + 31; step j of the chunk's eight mma
// takes its elements 4 j ... 4 j + 3.  A wide column's fragments are zero, its factor negative; returns
// whether one of the eight columns is wide.
template <bool kFp32>
__device__ __forceinline__ bool make_fragments(const Raw<kFp32>& raw, uint32_t (&b)[kFp32 ? 3 : 1][16], float& undo) {
    uint32_t top, least;
    range_of<kFp32>(raw, top, least);
    const uint32_t small = __ballot_sync(0xFFFFFFFFu, too_small<kFp32>(top, least));
    // 2^(14 - e) for a largest element in [2^e, 2^(e+1)), held to 2^126 so that its inverse is a
    // normal number; an infinity or a NaN among the elements stays one in fp16
    const int field = min(268 - (int)(top >> 23), 253);
    const float scale = __uint_as_float((uint32_t)field << 23);
    undo = __uint_as_float((uint32_t)(254 - field) << 23);
    if constexpr (kFp32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float lo = __uint_as_float(raw.words[2 * i]) * scale, hi = __uint_as_float(raw.words[2 * i + 1]) * scale;
#pragma unroll
            for (int part = 0; part < 3; ++part) {
                const __half2 h = __floats2half2_rn(lo, hi);
                b[part][i] = *reinterpret_cast<const uint32_t*>(&h);
                // what this part leaves over, exactly; nothing behind an infinity or a NaN
                const float2 f = __half22float2(h);
                lo = fabsf(f.x) <= 65504.0f ? (lo - f.x) * 2048.0f : 0.0f;
                hi = fabsf(f.y) <= 65504.0f ? (hi - f.y) * 2048.0f : 0.0f;
            }
        }
    } else {
        const uint32_t scale2 = (uint32_t)field << 7 | (uint32_t)field << 23;  // the power of two as a bf16 pair
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            uint32_t w;
            asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(raw.words[i]), "r"(scale2));
            const __half2 h = __floats2half2_rn(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
            b[0][i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    if (small >> (threadIdx.x & 28) & 15) {  // seldom
        undo = -1.0f;
#pragma unroll
        for (int part = 0; part < (kFp32 ? 3 : 1); ++part)
#pragma unroll
            for (int i = 0; i < 16; ++i) b[part][i] = 0;
    }
    return small != 0;
}

// The 16 bytes of codes (32 elements) and the scale bytes of one row that a lane decodes in one
// chunk.  A chunk or row behind the end is read as the last one instead, so that no load hangs on
// a branch: its activations are zero, or its sums are not stored.
struct Piece {
    uint4 codes;
    uint32_t scales;  // byte 0: elements 0..15 of the 32, byte 1: elements 16..31 (B = 32: byte 0 for all)
};

// kBytes aligned bytes, of which the first `there` exist; the others become zero
template <int kBytes>
__device__ __forceinline__ void copy_part_async(void* to, const uint8_t* from, int there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(kBytes),
                 "r"(there)
                 : "memory");
}

template <int kBytes>
__device__ __forceinline__ void copy_async(void* to, const uint8_t* from) {
    const uint32_t address = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(address), "l"(from) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(address), "l"(from), "n"(kBytes) : "memory");
}

// Rows that start anywhere.  Of an array of `bytes` bytes the aligned pieces that hold `count` rows' bytes from
// `column` on, a multiple of kSize: kPieces a row, neighbouring lanes side by side.  `row`, the first of
// the rows, and the others after it stand for row >> shift of the array.  What lies behind the array
// becomes zero.
template <int kSize, int kPieces>
__device__ __forceinline__ void copy_pieces(void* to, const uint8_t* array, int64_t bytes, int row_bytes, int shift, int row, int count,
                                            int column) {
    const int lane = threadIdx.x & 31;
    const int64_t start = (row >> shift) * (int64_t)row_bytes;
    const uint32_t off = (uint32_t)((uintptr_t)array + start) & (kSize - 1);
    const uint8_t* base = array + start - off;  // below the array for its first row if it does not start on a piece
    const int64_t left = bytes - start + off;   // from base on
    const bool inner = start >= off && left > (int64_t)count * row_bytes + column + kSize * kPieces;
    uint8_t* target = reinterpret_cast<uint8_t*>(to) + lane * kSize;
    int r = lane / kPieces, piece = lane % kPieces;
    for (int at = lane; at < count * kPieces; at += 32, target += 32 * kSize) {
        const uint32_t from = (((row + r >> shift) - (row >> shift)) * row_bytes + off & ~(kSize - 1u)) + column + kSize * piece;
        if (inner)
            copy_async<kSize>(target, base + from);
        else if (base + from < array)
            for (uint32_t e = 0; e < kSize; ++e) target[e] = e >= off && e < left ? base[e] : 0;
        else
            copy_part_async<kSize>(target, from < left ? base + from : base + kSize, from < left ? (int)min(left - from, (int64_t)kSize) : 0);
        r += 32 / kPieces, piece += 32 % kPieces;
        if (piece >= kPieces) piece -= kPieces, ++r;
    }
}

// The aligned pieces of 16 bytes that hold `wanted` of an array's bytes from `at` on, by one warp.
__device__ __forceinline__ void copy_run(uint4* to, const uint8_t* array, int64_t bytes, int64_t at, int wanted) {
    const int lane = threadIdx.x & 31, off = (int)((uintptr_t)(array + at) & 15);
    for (int piece = lane; piece * 16 < off + wanted; piece += 32) {
        const int64_t from = at - off + 16 * piece, left = bytes - from;
        if (from < 0)  // the first piece of an array that does not start on one
            for (int e = 0; e < 16; ++e) reinterpret_cast<uint8_t*>(to + piece)[e] = from + e >= 0 && e < left ? array[from + e] : 0;
        else if (left >= 16)
            copy_async<16>(to + piece, array + from);
        else
            copy_part_async<16>(to + piece, left > 0 ? array + from : array + at - off + 16, left > 0 ? (int)left : 0);
    }
}

// ... of the weight, for one chunk: nine pieces of 8 bytes of a row's codes, three of 4 of its scales
template <int kBlock>
__device__ __forceinline__ void copy_row_pieces(const Params& p, uint4* codes_to, uint4* scales_to, int row, int count, int chunk) {
    copy_pieces<8, 9>(codes_to, p.codes, p.rows * p.code_stride, (int)p.code_stride, 0, row, count, chunk * (kChunk / 2));
    copy_pieces<4, 3>(scales_to, p.scales, ((int64_t)(p.rows - 1 >> p.row_shift) + 1) * p.scale_stride, (int)p.scale_stride, p.row_shift,
                      row, count, chunk * (kChunk / kBlock));
}

// a lane's share of row `row` + r from there: the words shifted into place
template <int kBlock>
__device__ __forceinline__ Piece piece_of_row(const Params& p, const uint4* codes_from, const uint4* scales_from, int row, int r, int chunk) {
    const int c = threadIdx.x & 3;
    const uint32_t in_piece = (uint32_t)((uintptr_t)p.codes + (row + r) * p.code_stride) & 7, off = 8 * (in_piece & 3);
    const uint32_t* at = reinterpret_cast<const uint32_t*>(codes_from) + r * 18 + (in_piece >> 2) + 4 * c;
    const uint32_t scale_off = (uint32_t)((uintptr_t)p.scales + (row + r >> p.row_shift) * p.scale_stride + chunk * (kChunk / kBlock)) & 3;
    const uint8_t* scale_at = reinterpret_cast<const uint8_t*>(scales_from) + r * 12 + scale_off + c * (32 / kBlock);
    Piece piece;
    piece.codes = make_uint4(__funnelshift_r(at[0], at[1], off), __funnelshift_r(at[1], at[2], off),
                             __funnelshift_r(at[2], at[3], off), __funnelshift_r(at[3], at[4], off));
    piece.scales = kBlock == 16 ? scale_at[0] | (uint32_t)scale_at[1] << 8 : scale_at[0];
    return piece;
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// The scales of a lane's two rows (g and g + 8 of a 16-row tile) in one chunk, as fp16 pairs: [row][half]
template <int kBlock>
__device__ __forceinline__ void scale_pairs(const Piece (&piece)[2], uint32_t (&scale)[2][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        scale[h][0] = scale_half2(kBlock == 16 ? piece[h].scales & 0xFFu : piece[h].scales);
        scale[h][1] = kBlock == 16 ? scale_half2(piece[h].scales >> 8) : scale[h][0];
    }
}

// step j of the chunk's four: eight elements of each of the two rows
template <int kBlock>
__device__ __forceinline__ void decode(const Piece (&piece)[2], const uint32_t (&scale)[2][2], int j, uint32_t (&a)[2][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        e2m1x8_to_half2(word_of(piece[h].codes, j), a[h]);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[h][i] = mul_half2(a[h][i], scale[h][j / 2]);
    }
}

// The wide columns of one chunk, seldom needed.  What one warp reads for them: a chunk of eight tokens at most, and
// its codes and scales for up to kRowTiles times 16 rows.
template <bool kFp32, int kRowTiles>
struct Wide {
    Raw<kFp32> raw;
    Piece pieces[kRowTiles][2];
};

// 32 codes from `at` on, which may lie anywhere; what is not in the array counts as zero
__device__ __forceinline__ uint4 load_codes_anywhere(const uint8_t* at, const uint8_t* array, const uint8_t* end) {
    const uint32_t off = (uint32_t)(uintptr_t)at & 3;
    const uint8_t* aligned = at - off;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const uint8_t* from = aligned + 4 * i;
        w[i] = 0;
        if (from >= array && from + 4 <= end) {
            w[i] = __ldg(reinterpret_cast<const uint32_t*>(from));
        } else {
#pragma unroll 1
            for (int e = 0; e < 4; ++e)
                if (from + e >= array && from + e < end) w[i] |= (uint32_t)from[e] << (8 * e);
        }
    }
    return make_uint4(__funnelshift_r(w[0], w[1], 8 * off), __funnelshift_r(w[1], w[2], 8 * off), __funnelshift_r(w[2], w[3], 8 * off),
                      __funnelshift_r(w[3], w[4], 8 * off));
}

// ... of rows row0 ... row0 + row_count - 1, the last one again in the place of missing ones
template <bool kFp32, bool kVector, int kBlock, int kRowTiles>
__device__ __forceinline__ void load_pieces(const Params& p, Wide<kFp32, kRowTiles>& wide, int chunk, int row0, int row_count) {
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
#pragma unroll
    for (int tile = 0; tile < kRowTiles; ++tile)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Piece& piece = wide.pieces[tile][h];
            const int64_t row = row0 + min(16 * tile + g + 8 * h, row_count - 1);
            const uint8_t* codes = p.codes + row * p.code_stride + chunk * (kChunk / 2) + 16 * c;
            const uint8_t* scales = p.scales + (row >> p.row_shift) * p.scale_stride;
            const int at = chunk * (kChunk / kBlock) + c * (32 / kBlock);
            if constexpr (kVector) {
                piece.codes = __ldg(reinterpret_cast<const uint4*>(codes));
                piece.scales = kBlock == 16 ? __ldg(reinterpret_cast<const uint16_t*>(scales + at)) : __ldg(scales + at);
            } else {
                piece.codes = load_codes_anywhere(codes, p.codes, p.codes + p.rows * p.code_stride);
                piece.scales = at < p.scale_stride ? __ldg(scales + at) : 0;
                if (kBlock == 16 && at + 1 < p.scale_stride) piece.scales |= (uint32_t)__ldg(scales + at + 1) << 8;
            }
        }
}

// The wide columns' fragments: bf16; fp32 elements are cut off to 8 bits, not rounded, so that every rest is exact
// and 2^8 of it below twice the element.  Returns four bits for every token with a wide column.
template <bool kFp32>
__device__ __forceinline__ uint32_t make_wide_fragments(const Raw<kFp32>& raw, uint32_t (&b)[kFp32 ? 3 : 1][16]) {
    uint32_t top, least;
    range_of<kFp32>(raw, top, least);
    const uint32_t small = __ballot_sync(0xFFFFFFFFu, too_small<kFp32>(top, least));
    const bool wide = small >> (threadIdx.x & 28) & 15;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if constexpr (kFp32) {
            uint32_t lo = wide ? raw.words[2 * i] : 0, hi = wide ? raw.words[2 * i + 1] : 0;
#pragma unroll
            for (int part = 0; part < 3; ++part) {
                b[part][i] = lo >> 16 | (hi & 0xFFFF0000u);
                lo = __float_as_uint((__uint_as_float(lo) - __uint_as_float(lo & 0xFFFF0000u)) * 256.0f);
                hi = __float_as_uint((__uint_as_float(hi) - __uint_as_float(hi & 0xFFFF0000u)) * 256.0f);
            }
        } else {
            b[0][i] = wide ? raw.words[i] : 0;
        }
    }
    return small;
}

// ... times 16 rows, added to[token * stride + row]: a lane's tokens are 2 c and 2 c + 1, its rows g and g + 8
template <bool kFp32, int kBlock>
__device__ __forceinline__ void add_wide(const Piece (&now)[2], const uint32_t (&b)[kFp32 ? 3 : 1][16], uint32_t small, int row_count,
                                         float* to, int stride) {
    constexpr int kParts = kFp32 ? 3 : 1;
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
    uint32_t scale[2][2];
    scale_pairs<kBlock>(now, scale);
    float sum[kParts][4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t a[2][4];
        decode<kBlock>(now, scale, j, a);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // six significant bits, 2^-22 ... 2^16: exact in bf16
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[h][i]));
                a[h][i] = __float_as_uint(f.x) >> 16 | (__float_as_uint(f.y) & 0xFFFF0000u);
            }
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            mma_bf16(sum[part], a[0][0], a[1][0], a[0][1], a[1][1], b[part][4 * j], b[part][4 * j + 1]);
            mma_bf16(sum[part], a[0][2], a[1][2], a[0][3], a[1][3], b[part][4 * j + 2], b[part][4 * j + 3]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int token = 2 * c + (e & 1), row = g + 8 * (e >> 1);
        if (!(small >> (4 * token) & 15) || row >= row_count) continue;
        float whole = sum[0][e];
        if constexpr (kFp32) whole = __fmaf_rn(sum[kParts - 1][e], 0x1p-16f, __fmaf_rn(sum[kParts / 2][e], 0x1p-8f, whole));
        to[token * stride + row] += whole;
    }
}

__device__ __forceinline__ void store(const Params& p, int token, int64_t row, float value) {
    value *= p.factor;
    if (p.bias)
        value += p.bias_fp32 ? reinterpret_cast<const float*>(p.bias)[row]
                             : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[row]);
    const int64_t at = token * p.ldo + row;
    if (p.out_fp32)
        reinterpret_cast<float*>(p.out)[at] = value;
    else
        reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(value);
}

// Up to eight tokens.  kDepth: chunks that a warp keeps in registers.
template <bool kFp32, int kDepth, bool kVector, int kBlock>
__global__ void __launch_bounds__(kThreads, 1) packed_matvec_kernel(const Params p) {
    // the ring: kVector: [slot]{codes [chunk][row half][thread], scales [warp][chunk][row]}, otherwise [slot]{codes [row], scales [row]};
    // there one chunk of eight tokens' activations per warp as well, on its way to the lanes
    extern __shared__ uint4 ring[];
    constexpr int kSlot = kVector ? slot_pieces(kDepth) : kRowSlot;
    float* partial = reinterpret_cast<float*>(ring + kRing * kSlot + (kVector ? 0 : kStagePieces));  // [warp][token][row of the block]
    constexpr int kParts = kFp32 ? 3 : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int share = blockIdx.x % p.split, group = blockIdx.x / p.split, groups = gridDim.x / p.split;
    const int all_chunks = (p.k + kChunk - 1) / kChunk;
    const int first_chunk = all_chunks * share / p.split, chunks = all_chunks * (share + 1) / p.split;  // first and behind the last
    const int passes = max(1, (chunks - first_chunk + kWarps * kDepth - 1) / (kWarps * kDepth));
    const int first_row = (int)((int64_t)p.rows * group / groups);
    const int last_row = (int)((int64_t)p.rows * (group + 1) / groups);
    const int block_rows = p.rows_per_block;
    const int stride = (int)p.code_stride, scale_stride = (int)p.scale_stride;
    const int tokens = p.tokens;
    for (int row0 = first_row; row0 < last_row; row0 += block_rows) {
        const int row_count = min(block_rows, last_row - row0);
        const uint8_t* codes = p.codes + row0 * p.code_stride;
        const int scale_row0 = row0 >> p.row_shift;
        const uint8_t* scales = p.scales + scale_row0 * p.scale_stride;
        // Codes and scales of the tiles to come wait in a ring in shared memory, kRing - 1 tiles ahead.  Wide
        // rows: the codes in the slots of the lane that decodes them, the scale bytes of a row's chunk side
        // by side; others: a row of the tile per warp, its bytes of all warps' chunks in one run, for which the
        // CTA's warps wait for one another at every tile.  A row or chunk behind the end is not copied:
        // what its slot holds is finite, and meets zeros or is not stored.

        // the (pass, tile) that is copied next, and where this lane's first row of it lies
        int ahead_pass = 0, ahead_tile = 0;
        const uint8_t *ahead_codes = nullptr, *ahead_scales = nullptr;
        auto locate = [&]() {
            const int chunk = first_chunk + ahead_pass * kDepth * kWarps + warp;
            ahead_codes = codes + (int64_t)(ahead_tile + g) * stride + chunk * (kChunk / 2) + 16 * c;
            ahead_scales = scales + chunk * (kChunk / kBlock);
        };
        auto copy_ahead = [&](int slot) {
            if (!kVector && ahead_pass < passes) {
                const int chunk = first_chunk + ahead_pass * kWarps, here = min(kWarps, chunks - chunk);
                uint4* to = ring + slot * kSlot;
                const int64_t row = row0 + ahead_tile + warp;
                if (ahead_tile + warp < row_count) {
                    copy_run(to + warp * kRowPieces, p.codes, p.rows * p.code_stride, row * p.code_stride + chunk * (kChunk / 2),
                             here * (kChunk / 2));
                    copy_run(to + 16 * kRowPieces + warp * kRowScalePieces, p.scales,
                             ((int64_t)(p.rows - 1 >> p.row_shift) + 1) * p.scale_stride,
                             (row >> p.row_shift) * p.scale_stride + chunk * (kChunk / kBlock), here * (kChunk / kBlock));
                }
                ahead_tile += 16;
                if (ahead_tile >= row_count) ahead_tile = 0, ++ahead_pass;
            } else if (ahead_pass < passes) {
                uint4* to = ring + slot * kSlot + threadIdx.x;
                uint8_t* scales_to = reinterpret_cast<uint8_t*>(ring + slot * kSlot + kDepth * 2 * kThreads) + warp * kDepth * 128;
                const int row = ahead_tile + g + 8 * c;  // lanes 0 and 1 of a row bring the scales of it and the one 8 on
                const int scale_row = (row0 + row >> p.row_shift) - scale_row0;
#pragma unroll
                for (int d = 0; d < kDepth; ++d) {
                    if (first_chunk + (ahead_pass * kDepth + d) * kWarps + warp >= chunks) continue;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (ahead_tile + g + 8 * h < row_count)
                            copy_async<16>(to + (d * 2 + h) * kThreads, ahead_codes + h * 8 * stride + d * kWarps * (kChunk / 2));
                    if (c < 2 && row < row_count)
                        copy_async<kChunk / kBlock>(scales_to + d * 128 + (g + 8 * c) * (kChunk / kBlock),
                                                    ahead_scales + scale_row * scale_stride + d * kWarps * (kChunk / kBlock));
                }
                ahead_tile += 16;
                ahead_codes += 16 * stride;
                if (ahead_tile >= row_count) {
                    ahead_tile = 0, ++ahead_pass;
                    locate();
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int slot_now = 0;
        uint32_t wide = 0;  // bit i: this warp's i-th chunk has a wide column; bit 31: one of those from the 32nd on has
        if (kVector) locate();
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) copy_ahead(i);
        for (int pass = 0; pass < passes; ++pass) {
            uint32_t b[kDepth][kParts][16];
            float undo[kDepth][2];
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                const int chunk = first_chunk + (pass * kDepth + d) * kWarps + warp;
                float mine;
                const bool any = make_fragments<kFp32>(
                    kVector ? load_raw<kFp32>(p, g, g < tokens && chunk < chunks, chunk)
                            : load_staged<kFp32>(p, 0, chunk < chunks ? tokens : 0, chunk, reinterpret_cast<uint32_t*>(ring + kRing * kSlot) + warp * kStageWords),
                    b[d], mine);
                wide |= any ? 1u << min(pass * kDepth + d, 31) : 0;
                undo[d][0] = __shfl_sync(0xFFFFFFFFu, mine, 8 * c);
                undo[d][1] = __shfl_sync(0xFFFFFFFFu, mine, 8 * c + 4);
            }
            float* slot = partial + (warp * tokens + 2 * c) * block_rows + g;
#pragma unroll 2
            for (int tile = 0; tile < row_count; tile += 16, slot += 16) {
                Piece now[kDepth][2];
                if constexpr (kVector) {
                    __syncwarp();  // the slot that is filled now has been read
                    copy_ahead(slot_now == 0 ? kRing - 1 : slot_now - 1);
                    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
                    __syncwarp();  // scales come from other lanes
                    const uint4* from = ring + slot_now * kSlot + threadIdx.x;
                    const uint8_t* scales_from =
                        reinterpret_cast<const uint8_t*>(ring + slot_now * kSlot + kDepth * 2 * kThreads) + warp * kDepth * 128;
#pragma unroll
                    for (int d = 0; d < kDepth; ++d)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            now[d][h].codes = from[(d * 2 + h) * kThreads];
                            const uint8_t* at = scales_from + d * 128 + (g + 8 * h) * (kChunk / kBlock) + c * (32 / kBlock);
                            now[d][h].scales = kBlock == 16 ? *reinterpret_cast<const uint16_t*>(at) : *at;
                        }
                } else {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
                    __syncthreads();  // all copies of this tile are there, and the slot before has been read
                    copy_ahead(slot_now == 0 ? kRing - 1 : slot_now - 1);
                    const uint4* from = ring + slot_now * kSlot;
                    const int chunk = first_chunk + pass * kWarps;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = g + 8 * h;
                        const int64_t row = row0 + tile + r;
                        const uint32_t off = (uint32_t)((uintptr_t)p.codes + row * p.code_stride) & 15;
                        const uint32_t* at = reinterpret_cast<const uint32_t*>(from + r * kRowPieces) + (off >> 2) + warp * 16 + 4 * c;
                        const uint32_t scale_off =
                            (uint32_t)((uintptr_t)p.scales + (row >> p.row_shift) * p.scale_stride + chunk * (kChunk / kBlock)) & 15;
                        const uint8_t* scale_at = reinterpret_cast<const uint8_t*>(from + 16 * kRowPieces + r * kRowScalePieces) + scale_off +
                                                  warp * (kChunk / kBlock) + c * (32 / kBlock);
                        const uint32_t turn = 8 * (off & 3);
                        now[0][h].codes = make_uint4(__funnelshift_r(at[0], at[1], turn), __funnelshift_r(at[1], at[2], turn),
                                                     __funnelshift_r(at[2], at[3], turn), __funnelshift_r(at[3], at[4], turn));
                        now[0][h].scales = kBlock == 16 ? scale_at[0] | (uint32_t)scale_at[1] << 8 : scale_at[0];
                    }
                }
                slot_now = slot_now == kRing - 1 ? 0 : slot_now + 1;
                float total[4];
#pragma unroll
                for (int d = 0; d < kDepth; ++d) {
                    float sum[kParts][4] = {};
                    uint32_t scale[2][2];
                    scale_pairs<kBlock>(now[d], scale);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a[2][4];
                        decode<kBlock>(now[d], scale, j, a);
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            const uint32_t(&x)[16] = b[d][part];
                            mma_f16(sum[part], a[0][0], a[1][0], a[0][1], a[1][1], x[4 * j], x[4 * j + 1]);
                            mma_f16(sum[part], a[0][2], a[1][2], a[0][3], a[1][3], x[4 * j + 2], x[4 * j + 3]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float whole = sum[0][i];
                        if constexpr (kFp32)
                            whole = __fmaf_rn(sum[2][i], 0x1p-22f, __fmaf_rn(sum[1][i], 0x1p-11f, whole));
                        total[i] = d == 0 ? whole * undo[d][i & 1] : __fmaf_rn(whole, undo[d][i & 1], total[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (2 * c + i < tokens) {
                        float* at = slot + i * block_rows;
                        if (pass > 0) {
                            total[i] += at[0];
                            total[i + 2] += at[8];
                        }
                        at[0] = total[i];
                        at[8] = total[i + 2];
                    }
            }
        }
        // wide columns, seldom: chunk by chunk of this warp's that has some, 64 rows at a time
        for (int turn = 0; wide; ++turn) {
            if (turn < 31 && !(wide & 1)) {
                wide >>= 1;
                continue;
            }
            const int chunk = first_chunk + turn * kWarps + warp;
            if (chunk >= chunks) break;
            if (turn < 31) wide >>= 1;  // the last bit stands for all further ones
            uint32_t b[kParts][16];
            Wide<kFp32, 4> now;
            load_pieces<kFp32, kVector, kBlock, 4>(p, now, chunk, row0, row_count);
            const uint32_t small = make_wide_fragments<kFp32>(load_raw<kFp32>(p, g, g < tokens, chunk), b);
#pragma unroll 1
            for (int r = 0; r < row_count; r += 64) {
                if (r > 0) load_pieces<kFp32, kVector, kBlock, 4>(p, now, chunk, row0 + r, row_count - r);
#pragma unroll
                for (int tile = 0; tile < 4; ++tile)
                    if (r + 16 * tile < row_count)
                        add_wide<kFp32, kBlock>(now.pieces[tile], b, small, row_count - r - 16 * tile,
                                                partial + warp * tokens * block_rows + r + 16 * tile, block_rows);
            }
        }
        __syncthreads();
        if (p.split > 1) {
            // the sums of this CTA's warps, in the place of its first warp's; then those of the cluster
            for (int i = threadIdx.x; i < row_count * tokens; i += kThreads) {
                const int token = i / row_count, r = i - token * row_count;
                float value = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) value += partial[(w * tokens + token) * block_rows + r];
                partial[token * block_rows + r] = value;
            }
            cooperative_groups::this_cluster().sync();
        }
        for (int i = share * kThreads + threadIdx.x; i < row_count * tokens; i += p.split * kThreads) {
            const int token = i / row_count, r = i - token * row_count;
            float value = 0.0f;
            if (p.split > 1) {
                for (int q = 0; q < p.split; ++q)
                    value += cooperative_groups::this_cluster().map_shared_rank(partial, q)[token * block_rows + r];
            } else {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) value += partial[(w * tokens + token) * block_rows + r];
            }
            store(p, token, row0 + r, value);
        }
        if (p.split > 1)
            cooperative_groups::this_cluster().sync();  // the others have read this CTA's sums
        else
            __syncthreads();
    }
}

template <bool kFp32, int kDepth, bool kVector, int kBlock>
int launch_few(Params p, cudaStream_t stream) {
    constexpr size_t kRingBytes = (kVector ? kRing * slot_pieces(kDepth) : kRing * kRowSlot + kStagePieces) * sizeof(uint4);
    constexpr auto kKernel = packed_matvec_kernel<kFp32, kDepth, kVector, kBlock>;
    cudaError_t error = allow_shared<kKernel>((int)kRingBytes + kPartialFloats * 4);
    if (error != cudaSuccess) return record_cuda_error(error);
    // A long reduction axis and not many rows: with the rows spread over all SMs, every one of them would convert
    // all activations, for a few row tiles each time.  Pairs of CTAs share the axis and own twice the rows
    // (8 x 4096 x 21504: 23.2 -> 20.1 us; four CTAs 22.0, since only 33 such clusters fit on the SMs).
    const int passes = (p.k + kChunk * kWarps * kDepth - 1) / (kChunk * kWarps * kDepth);
    p.split = passes > 1 && p.rows <= 64 * sm_count() ? 2 : 1;
    int grid = sm_count();
    if (p.split > 1) {
        grid = resident_clusters<kKernel>(p.split, kThreads, (int)kRingBytes + kPartialFloats * 4);
        if (grid <= 0) grid = sm_count(), p.split = 1;
    }
    if (grid > p.rows) grid = p.rows;
    const int own = (p.rows + grid - 1) / grid;
    int block = kPartialFloats / (kWarps * p.tokens) / 16 * 16;
    const int need = (own + 15) / 16 * 16;
    if (block > need) block = need;
    p.rows_per_block = block;
    const size_t bytes = kRingBytes + (size_t)kWarps * p.tokens * block * sizeof(float);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid * p.split);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = p.split;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = p.split > 1 ? 1 : 0;
    return record_cuda_error(cudaLaunchKernelEx(&config, kKernel, p));
}

// ---- more than eight tokens ---------------------------------------------------------------------

constexpr int kManyWarps = 8;     // four times 32 rows, for each of two halves of the CTA's chunks
constexpr int kManyThreads = kManyWarps * 32;
constexpr int kManyRows = 128;
constexpr int kManyPad = kManyRows + 4;  // rows of a token's sums: the lanes of a fragment meet no bank twice
constexpr int kManyRing = 3;                // chunks on their way per half, one of them in use
// 16-byte pieces of 32 rows' codes of a chunk and their scales.  Wide rows: 64 and 8 bytes a row; others: the
// aligned pieces that hold them, nine of 8 bytes and three of 4.
__host__ __device__ constexpr int many_slot(bool vector) { return vector ? 2 * 2 * 32 + 16 : 32 * (9 * 8 + 3 * 4) / 16; }
// ... and of a chunk's activations: fragments, and the factors behind them
__host__ __device__ constexpr int many_stage(int tiles, int parts) { return tiles * (parts * 128 + 2); }

// The activations as the product reads them: [chunk][tile of 8 tokens][part][step][lane] 16 bytes, and
// the factors that undo the chunks' powers of two: [chunk][tile][token], and a byte that tells whether a column is
// wide: [chunk][tile].  One warp per chunk and tile.
template <bool kFp32>
__global__ void __launch_bounds__(kManyThreads) prepare_kernel(const Params p, uint4* fragments, float* undo, uint8_t* wide, int chunks, int tiles) {
    constexpr int kParts = kFp32 ? 3 : 1;
    __shared__ uint4 stage[kManyWarps * kStageWords / 4];
    launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int64_t unit = (int64_t)blockIdx.x * kManyWarps + warp;
    const int chunk = (int)(unit / tiles), tile = (int)(unit % tiles);
    if (chunk >= chunks) return;
    const int here = min(8, p.tokens - 8 * tile);
    uint32_t b[kParts][16];
    float mine;
    const bool any =
        make_fragments<kFp32>(p.vector_x ? load_raw<kFp32>(p, 8 * tile + g, g < here, chunk)
                                         : load_staged<kFp32>(p, 8 * tile, here, chunk, reinterpret_cast<uint32_t*>(stage) + warp * kStageWords),
                              b, mine);
    uint4* to = fragments + unit * (kParts * 128) + lane;
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            to[part * 128 + j * 32] = make_uint4(b[part][4 * j], b[part][4 * j + 1], b[part][4 * j + 2], b[part][4 * j + 3]);
    if (c == 0) undo[unit * 8 + g] = mine;
    if (lane == 0) wide[unit] = any;
}

// What a warp of the product owns: rows row0 ... of its CTA's block, every second chunk from `first` to before
// `last`, tiles tile0 ... tile0 + here - 1.
struct Share {
    int block_row, own, row0, row_count, tile0, here, half, first, last;
};

template <int kTiles>
__device__ __forceinline__ Share share_of(const Params& p, int chunks, int tiles, int block, int warp) {
    Share s;
    const int share = block % p.split, place = block / p.split;
    // groups of tokens, as even as their number allows (72 x 4096 x 4096: 26.8 -> 22.1 us); those of a block of
    // rows start side by side
    const int groups = (tiles + kTiles - 1) / kTiles, each = (tiles + groups - 1) / groups;
    const int row_block = place / groups;
    s.tile0 = place % groups * each;
    s.block_row = (int)((int64_t)p.rows * row_block / p.row_blocks);
    s.own = (int)((int64_t)p.rows * (row_block + 1) / p.row_blocks) - s.block_row;  // kManyRows at most
    s.here = min(each, tiles - s.tile0);
    s.row0 = s.block_row + warp % 4 * 32;
    s.half = warp / 4;
    s.first = (int)((int64_t)chunks * share / p.split) + s.half;
    s.last = (int)((int64_t)chunks * (share + 1) / p.split);
    s.row_count = min(32, s.own - warp % 4 * 32);
    return s;
}

// The block's and the thread's index, read again: what follows from them is computed again, not kept.
__device__ __forceinline__ int block_index_again() {
    int v;
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(v));
    return v;
}
__device__ __forceinline__ int thread_index_again() {
    int v;
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(v));
    return v;
}

template <bool kFp32, int kTiles, bool kVector, int kBlock>
__global__ void __launch_bounds__(kManyThreads, kFp32 || kTiles > 4 ? 1 : 2)
    packed_matmul_kernel(const Params p, const uint4* fragments, const float* undo, const uint8_t* wide, int chunks, int tiles) {
    constexpr int kParts = kFp32 ? 3 : 1;
    constexpr int kStage = many_stage(kTiles, kParts);
    // activations [half][slot], then, kVector, codes and scales [warp][slot]; afterwards the sums [half][token][row]
    extern __shared__ uint4 ring[];
    constexpr int kSlot = many_slot(kVector);
    float* partial = reinterpret_cast<float*>(ring);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const Share mine = share_of<kTiles>(p, chunks, tiles, blockIdx.x, warp);
    const int share = blockIdx.x % p.split, tile0 = mine.tile0, block_row = mine.block_row, own = mine.own, here = mine.here,
              row0 = mine.row0, half = mine.half, first = mine.first, row_count = mine.row_count;
    const int count = mine.last > first ? (mine.last - first + 1) / 2 : 0;
    const bool active = row_count > 0;
    const int stride = (int)p.code_stride, scale_stride = (int)p.scale_stride;
    const uint8_t* codes = p.codes + row0 * p.code_stride;
    const int scale_row0 = row0 >> p.row_shift;
    const uint8_t* scales = p.scales + scale_row0 * p.scale_stride;

    // codes and scales of the chunks to come: wide rows as in the kernel for few tokens, with the scales of
    // a row per lane; others in aligned pieces of 8 and 4 bytes
    uint4* slots = ring + 2 * kManyRing * kStage + warp * kManyRing * kSlot;
    auto copy_codes = [&](int i) {
        if (i < count && active) {
            const int chunk = first + 2 * i;
            uint4* to = slots + i % kManyRing * kSlot;
            if constexpr (!kVector) {
                copy_row_pieces<kBlock>(p, to, to + 32 * 9 / 2, row0, row_count, chunk);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = 8 * q + g;
                    if (row < row_count) copy_async<16>(to + q * 32 + lane, codes + row * stride + chunk * (kChunk / 2) + 16 * c);
                }
                if (lane < row_count)
                    copy_async<kChunk / kBlock>(reinterpret_cast<uint8_t*>(to + 128) + lane * 8,
                                                scales + ((row0 + lane >> p.row_shift) - scale_row0) * scale_stride + chunk * (kChunk / kBlock));
            }
        }
    };
    // the chunks' activations, by the four warps that use them
    uint4* stages = ring + half * kManyRing * kStage;
    auto copy_activations = [&](int i) {
        if (i < count) {
            const int64_t unit = (int64_t)(first + 2 * i) * tiles + tile0;
            uint4* to = stages + i % kManyRing * kStage;
            const uint4* from = fragments + unit * (kParts * 128);
            for (int at = threadIdx.x & 127; at < here * kParts * 128; at += 128)
                copy_async<16>(to + at, reinterpret_cast<const uint8_t*>(from + at));
            if ((threadIdx.x & 127) < here * 2)
                copy_async<16>(to + kTiles * kParts * 128 + (threadIdx.x & 127),
                               reinterpret_cast<const uint8_t*>(undo + unit * 8 + (threadIdx.x & 127) * 4));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kManyRing - 1; ++i) copy_codes(i);
    wait_for_launcher();  // the activations are prepared
#pragma unroll
    for (int i = 0; i < kManyRing - 1; ++i) copy_activations(i);

    uint32_t signs = 0;  // of the factors: that of a wide column is negative
    float total[2][kTiles][4] = {};
    for (int i = 0; i < count; ++i) {
        // this thread's copies for chunk i are there; behind the barrier all are, and the slot before is free
        asm volatile("cp.async.wait_group %0;" ::"n"(kManyRing - 2) : "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
        copy_codes(i + kManyRing - 1);
        copy_activations(i + kManyRing - 1);
        if (!active) continue;
        Piece now[2][2];
        if constexpr (kVector) {
            const uint4* from = slots + i % kManyRing * kSlot;
            const uint8_t* scales_from = reinterpret_cast<const uint8_t*>(from + 128) + g * 8 + c * (32 / kBlock);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                now[q / 2][q % 2].codes = from[q * 32 + lane];
                const uint8_t* at = scales_from + q * 64;
                now[q / 2][q % 2].scales = kBlock == 16 ? *reinterpret_cast<const uint16_t*>(at) : *at;
            }
        } else {
            const uint4* slot = slots + i % kManyRing * kSlot;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                now[q / 2][q % 2] = piece_of_row<kBlock>(p, slot, slot + 32 * 9 / 2, row0, 8 * q + g, first + 2 * i);
        }
        const uint4* from = stages + i % kManyRing * kStage + lane;
        const float2* undo_from = reinterpret_cast<const float2*>(from - lane + kTiles * kParts * 128) + c;
        uint32_t scale[2][2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) scale_pairs<kBlock>(now[r], scale[r]);
        float sum[2][kTiles][kParts][4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a[2][2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) decode<kBlock>(now[r], scale[r], j, a[r]);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                if (t % 2 == 0 && t >= here) break;  // a tile behind the last one: sums that are not stored
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    const uint4 x = from[(t * kParts + part) * 128 + j * 32];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        mma_f16(sum[r][t][part], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], x.x, x.y);
                        mma_f16(sum[r][t][part], a[r][0][2], a[r][1][2], a[r][0][3], a[r][1][3], x.z, x.w);
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (t % 2 == 0 && t >= here) break;
            const float2 back = undo_from[t * 4];
            if (t < here) signs |= __float_as_uint(back.x) | __float_as_uint(back.y);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float whole = sum[r][t][0][e];
                    if constexpr (kFp32)
                        whole = __fmaf_rn(sum[r][t][kParts - 1][e], 0x1p-22f, __fmaf_rn(sum[r][t][kParts / 2][e], 0x1p-11f, whole));
                    total[r][t][e] = __fmaf_rn(whole, e & 1 ? back.y : back.x, total[r][t][e]);
                }
        }
    }

    __syncthreads();  // the ring's memory takes the sums
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                partial[(half * kTiles * 8 + 8 * t + 2 * c + (e & 1)) * kManyPad + warp % 4 * 32 + 16 * r + g + 8 * (e >> 1)] = total[r][t][e];
    if (__any_sync(0xFFFFFFFFu, signs >> 31)) {
        // wide columns, seldom: 32 of the half's chunks at a time, each lane looks at one; then one unit (chunk and tile)
        // after the other, the next one's reads in flight
        const Share again = share_of<kTiles>(p, chunks, tiles, block_index_again(), thread_index_again() >> 5);
        float* sums = partial + again.half * kTiles * 8 * kManyPad + again.row0 - again.block_row;
#pragma unroll 1
        for (int base = again.first; base < again.last && again.row_count > 0; base += 64) {
            const int mine = base + 2 * lane;
            uint32_t bits = 0;  // of the tiles of this lane's chunk
            if (mine < again.last)
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    if (t < again.here && __ldcg(wide + (int64_t)mine * tiles + again.tile0 + t)) bits |= 1u << t;
            auto next = [&]() {  // a unit that is left: lane * 8 + tile, or -1
                const uint32_t left = __ballot_sync(0xFFFFFFFFu, bits != 0);
                if (left == 0) return -1;
                const int from = __ffs(left) - 1, t = __ffs(__shfl_sync(0xFFFFFFFFu, bits, from)) - 1;
                if (lane == from) bits &= bits - 1;
                return from * 8 + t;
            };
            Wide<kFp32, 2> now, then;
            auto load = [&](Wide<kFp32, 2>& unit, int at) {
                const int chunk = base + 2 * (at / 8), token = 8 * (again.tile0 + at % 8);
                load_pieces<kFp32, kVector, kBlock, 2>(p, unit, chunk, again.row0, again.row_count);
                unit.raw = load_raw<kFp32>(p, token + g, token + g < p.tokens, chunk);
            };
            int at = next();
            if (at >= 0) load(now, at);
#pragma unroll 1
            while (at >= 0) {
                const int following = next();
                if (following >= 0) load(then, following);
                uint32_t b[kParts][16];
                const uint32_t small = make_wide_fragments<kFp32>(now.raw, b);
#pragma unroll
                for (int tile = 0; tile < 2; ++tile)
                    add_wide<kFp32, kBlock>(now.pieces[tile], b, small, again.row_count - 16 * tile,
                                            sums + at % 8 * 8 * kManyPad + 16 * tile, kManyPad);
                now = then;
                at = following;
            }
        }
    }
    __syncthreads();
    const int tokens = min(here * 8, p.tokens - tile0 * 8);
    constexpr int kOther = kTiles * 8 * kManyPad;  // the second half's sums
    if (p.split > 1) {
        for (int i = threadIdx.x; i < kManyRows * tokens; i += kManyThreads) {
            float* at = partial + i / kManyRows * kManyPad + i % kManyRows;
            *at += at[kOther];
        }
        cooperative_groups::this_cluster().sync();
    }
    for (int i = share * kManyThreads + threadIdx.x; i < kManyRows * tokens; i += p.split * kManyThreads) {
        const int token = i / kManyRows, row = i % kManyRows, at = token * kManyPad + row;
        if (row >= own) continue;
        float value = 0.0f;
        if (p.split > 1) {
            for (int q = 0; q < p.split; ++q) value += cooperative_groups::this_cluster().map_shared_rank(partial, q)[at];
        } else {
            value = partial[at] + partial[at + kOther];
        }
        store(p, tile0 * 8 + token, block_row + row, value);
    }
    if (p.split > 1) cooperative_groups::this_cluster().sync();  // the others have read this CTA's sums
}

// bytes of the prepared activations: fragments, factors and the bytes of wide columns
size_t workspace_of(bool fp32, int64_t tokens, int64_t cols) {
    if (tokens <= kFewTokens) return 0;
    const size_t units = (size_t)((cols + kChunk - 1) / kChunk) * ((tokens + 7) / 8);
    return units * ((fp32 ? 3 : 1) * 2048 + 32 + 1);
}

template <bool kFp32, int kTiles, bool kVector, int kBlock>
int launch_many(Params p, void* workspace, cudaStream_t stream) {
    constexpr auto kKernel = packed_matmul_kernel<kFp32, kTiles, kVector, kBlock>;
    constexpr int kSums = 2 * kTiles * 8 * kManyPad * 4,
                  kRingBytes = (2 * many_stage(kTiles, kFp32 ? 3 : 1) + kManyWarps * many_slot(kVector)) * kManyRing * 16;
    constexpr int kBytes = kSums > kRingBytes ? kSums : kRingBytes;
    cudaError_t error = allow_shared<kKernel>(kBytes);
    if (error != cudaSuccess) return record_cuda_error(error);
    const int chunks = (p.k + kChunk - 1) / kChunk, tiles = (p.tokens + 7) / 8;
    const int64_t row_blocks = (p.rows + kManyRows - 1) / kManyRows, groups = (tiles + kTiles - 1) / kTiles;
    // What does not fill the SMs' last turn is spread over it (16 x 21504 x 4096: 168 blocks of 128 rows
    // 33.4 us, 296 of 73 rows 31.9); fewer blocks of rows than they have room for: clusters share the
    // reduction axis (33 x 4096 x 4096 takes four CTAs a block).
    const int64_t room = sm_count() * (kFp32 || kTiles > 4 ? 1 : 2), turns = (row_blocks * groups + room - 1) / room;
    p.row_blocks = (int)row_blocks;
    p.split = (int)(room / (row_blocks * groups));
    if (p.split < 2 && room * turns / groups > row_blocks) p.row_blocks = (int)(room * turns / groups);
    if (p.row_blocks > p.rows) p.row_blocks = p.rows;
    p.split = p.split < 1 ? 1 : p.split > 8 ? 8 : p.split;
    if (p.split > (chunks + 3) / 4) p.split = (chunks + 3) / 4;
    const int64_t places = p.row_blocks * groups;
    // ... as many as can run at a time: clusters do not straddle the SMs' groups (39 x 2923 x 6181 in fp32, 46
    // blocks: clusters of three 58 us, of two 55)
    while (p.split > 1 && places > resident_clusters<kKernel>(p.split, kManyThreads, kBytes)) --p.split;
    const int64_t units = (int64_t)chunks * tiles;
    if (places > 0x7FFFFFFF / 8 || units > (int64_t)0x7FFFFFFF * kManyWarps) {
        record_error_text("more rows times tokens than one launch covers");
        return UE5M3_ERR_TOO_LARGE;
    }
    uint4* fragments = reinterpret_cast<uint4*>(workspace);
    float* undo = reinterpret_cast<float*>(fragments + units * (kFp32 ? 384 : 128));
    uint8_t* wide = reinterpret_cast<uint8_t*>(undo + units * 8);
    prepare_kernel<kFp32><<<(unsigned)((units + kManyWarps - 1) / kManyWarps), kManyThreads, 0, stream>>>(p, fragments, undo, wide, chunks, tiles);
    const int status = check_launch();
    if (status != UE5M3_OK) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(places * p.split));
    config.blockDim = dim3(kManyThreads);
    config.dynamicSmemBytes = kBytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = p.split;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = p.split > 1 ? 2 : 1;
    return record_cuda_error(cudaLaunchKernelEx(&config, kKernel, p, (const uint4*)fragments, (const float*)undo, (const uint8_t*)wide, chunks, tiles));
}

template <bool kVector, int kBlock>
int dispatch(const Params& p, bool fp32, void* workspace, cudaStream_t s) {
    if (p.tokens <= kFewTokens)
        return fp32 ? launch_few<true, 1, kVector, kBlock>(p, s) : launch_few<false, kVector ? 2 : 1, kVector, kBlock>(p, s);
    // 32 tokens at a time leave registers for two CTAs on an SM, 64 read the weight once: 60 x 2718 x 15360
    // 30.3 us against 31.3, 33 x 4096 x 4096 13.5 against 16.5, and 64 x 300 x 4096 10.6 against 8.3.
    if (fp32) return launch_many<true, 4, kVector, kBlock>(p, workspace, s);
    return p.tokens <= 32 ? launch_many<false, 4, kVector, kBlock>(p, workspace, s) : launch_many<false, 8, kVector, kBlock>(p, workspace, s);
}

}  // namespace matvec
}  // namespace ue5m3

extern "C" size_t ue5m3_packed_matvec_workspace_bytes(int x_dtype, int64_t tokens, int64_t cols) {
    return tokens > 0 && cols > 0 ? ue5m3::matvec::workspace_of(x_dtype == UE5M3_DTYPE_FP32, tokens, cols) : 0;
}

extern "C" int ue5m3_packed_matvec(const void* x, int x_dtype, int64_t tokens, int64_t ldx, const uint8_t* codes,
                                   const uint8_t* scales, int64_t rows, int64_t cols, int block, int two_d, float dec,
                                   const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    using namespace ue5m3;
    if (!x || !codes || !scales || !out || tokens <= 0 || rows <= 0 || cols <= 0 || ldx < cols || ldo < rows)
        return UE5M3_ERR_INVALID_ARGUMENT;
    if ((x_dtype | out_dtype | bias_dtype) & ~1) return UE5M3_ERR_INVALID_ARGUMENT;
    if (block != 16 && block != 32) return UE5M3_ERR_BLOCK_SIZE;
    if (tokens > (1 << 24) || rows > (1 << 30) || cols > (1 << 22)) {
        record_error_text("at most 2^24 tokens, 2^30 rows and 2^22 columns");
        return UE5M3_ERR_TOO_LARGE;
    }
    const bool fp32 = x_dtype == UE5M3_DTYPE_FP32;
    const int element = fp32 ? 4 : 2;
    if ((uintptr_t)x % element || (uintptr_t)out % (out_dtype == UE5M3_DTYPE_FP32 ? 4 : 2) ||
        (bias && (uintptr_t)bias % (bias_dtype == UE5M3_DTYPE_FP32 ? 4 : 2)))
        return UE5M3_ERR_ALIGNMENT;
    const size_t need = matvec::workspace_of(fp32, tokens, cols);
    if (need > 0 && (!workspace || workspace_bytes < need)) return UE5M3_ERR_SCRATCH;
    if (need > 0 && (uintptr_t)workspace % 16) return UE5M3_ERR_ALIGNMENT;
    matvec::Params p;
    p.x = x;
    p.ldx = ldx;
    p.codes = codes;
    p.scales = scales;
    p.bias = bias;
    p.out = out;
    p.ldo = ldo;
    p.code_stride = (cols + 1) / 2;
    p.scale_stride = (cols + block - 1) / block;
    p.tokens = (int)tokens;
    p.rows = (int)rows;
    p.k = (int)cols;
    p.row_shift = !two_d ? 0 : block == 16 ? 4 : 5;
    // whole chunks of codes and scales, copied asynchronously
    const bool vector = cols % matvec::kChunk == 0 && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 8 == 0;
    p.vector_x = (uintptr_t)x % 16 == 0 && (ldx * element) % 16 == 0;
    p.bias_fp32 = bias_dtype == UE5M3_DTYPE_FP32;
    p.out_fp32 = out_dtype == UE5M3_DTYPE_FP32;
    p.factor = 16.0f * dec;
    cudaStream_t s = (cudaStream_t)stream;
    if (block == 16) return vector ? matvec::dispatch<true, 16>(p, fp32, workspace, s) : matvec::dispatch<false, 16>(p, fp32, workspace, s);
    return vector ? matvec::dispatch<true, 32>(p, fp32, workspace, s) : matvec::dispatch<false, 32>(p, fp32, workspace, s);
}
