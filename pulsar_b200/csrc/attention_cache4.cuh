// Attention over keys and values held in 4 bits (cache4.cuh has the format).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  over the keys j that a query at position p sees: j <= p, and j > p - window
//
// A query token at place t of the n that its sequence brings stands at position kv_len - n + t; with cu_q null every sequence brings one.
// Keys whose page is not one of the pool are not seen.  A query that sees nothing gives zeros.
//
// With k = m + s c and v = m' + s' c' for a group g of 32 channels, both products work on the codes themselves:
//
//   q.k_j = sum_g s_jg (sum_{i in g} q_i c_ji) + m_jg (sum_{i in g} q_i)          v: sum_j (p_j s'_jg) c'_ji + sum_j p_j m'_jg
//
// A code becomes an operand by one logical instruction for two of them.  Keys are taken in float16, where the bits of c alone are c 2^-24 and
// those of c << 4 are c 2^-20 (the products take subnormal numbers as they are), with q scaled to float16 by a power of two a row.  Values are taken in
// bfloat16, whose range a weight times a step needs: 128 + c is the bits 0x4300 | c.  A block takes one sequence, kv head,
// up to 8 NT rows (query heads of the kv head, tokens) and a part of the keys; its warps take runs of 32 keys in turn, each through
// buffers of its own in shared memory, so that nobody waits for anybody until the end.  mma.sync m16n8k16 has the keys in its 16 rows for
// the scores and the channels for the weighted sum, and the rows of the block in its 8 columns, where rows in its 16 would be mostly empty.
// Where a head has an even number of groups, 4 rows (2) stand in 8 columns twice (four times), and a copy of a row takes every second (fourth) group:
// no lane computes for an empty column what belongs to a group, key and column, and a 32-bit word of codes, whose halves are two
// neighbouring groups, is an operand as it is: its halves stand in two places of the sum, of which each copy's other operand has one empty.
// The weights change places between the two products by movmatrix.
//
// What bounds it: the latency of a turn, one chain of products, shuffles, exponentials and products.  4 query heads a kv head, heads of 128, bfloat16: 317 warp
// instructions for 16 keys (a third of them shifts and masks of codes, 18 products) fill 54 % of the issue slots with the three blocks an SM that registers
// allow, 10.6 warps, ALU 51, products 24, and it takes the same time when all pages lie in L2.  64 sequences of 4,096 to 8,192 keys take 108 us (507 MB: 4.7 TB/s; keys beyond the first thousands come at 5.4), 8 of 4,096 take
// 17, one of 900 takes 5.5.  16 rows of a block take 588 instructions for 16 keys, less than twice as many for four times the
// rows: 12 portions of 7 tokens over 1,300 to 2,600 keys take 39 us.  (tcgen05 would want codes as bfloat16 in shared memory, which is more traffic there
// than all the rest.  Tried: keys and values refilled apart, 111 us instead of 108 at the time; four blocks of two buffers an SM, 111; five warps a block, 145;
// copies of columns for 8 and 16 rows too, 56 instead of 44 for the portions.)
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "cache4.cuh"
#include "mma_common.cuh"

namespace pb {

constexpr int kTile4 = 32;              // keys of a warp's turn: two halves of 16
constexpr int kWarps4 = 4;
constexpr int kFold4 = 4;               // turns after which values' offsets are taken off (a power of two)
constexpr float kLowest4 = -3.0e38f;    // a running maximum before the first key

struct Attend4 {
    const void* q;
    void* out;
    Pool4 k, v;
    float* sums;                        // [blocks, 2, rows of a block, D] weighted sums, behind them [.., 2] maxima and sums of weights
    int* plan;                          // turns of a block, then where the turns of every entry begin
    const int* table;
    const int* kv_len;
    const int* cu_q;                    // null: one token each
    int width, n_rows, n_seqs, Hq, Hkv, page_size, page_shift, n_pages, row_blocks;     // row_blocks: entries of a sequence
    int blocks;                         // of even shares; below 0: clusters of -blocks
    int window;
    float scale_log2;
    PoolBounds bounds;
};

// The work is dealt out in turns of 32 keys.  An entry is a sequence and as many of its rows (tokens times the query heads of a kv head) as a block
// takes; what the lengths are is read here, on the device: a captured call serves any.  Either an entry and kv head is a cluster's, whose blocks take
// equal parts (attend_4bit_cluster_kernel); or the turns of all entries, kv head by kv head, stand in one line, and every block takes a run of the
// line of the same length (attend_4bit_kernel, then join_4bit_kernel).  Which of them: pb_attention_4bit_blocks.  Two ways to lay the line out,
// whichever ends sooner:
//   apart    every head begins with a block of its own, and its last block may have less: few heads, as many blocks as there are
//   packed   a head follows the other, with a gap of kGap4 turns between them that stands for what it costs to begin and end one
// In either a block has at most one head that another one began and one that another one ends.
struct Entry4 {
    int seq, first_token, n_tokens, kv_len, row0, token0, token1;
    int first, last, turns;             // the keys [first, last] that any of its rows sees; turns begin at first rounded down

    __device__ __forceinline__ Entry4(const Attend4& a, int entry, int rows) : Entry4(a, entry / a.row_blocks, entry % a.row_blocks, rows) {}
    __device__ __forceinline__ Entry4(const Attend4& a, int sequence, int row_block, int rows) {
        const int group = a.Hq / a.Hkv;
        seq = sequence;
        row0 = row_block * rows;
        first_token = a.cu_q ? a.cu_q[seq] : seq;
        n_tokens = a.cu_q ? a.cu_q[seq + 1] - first_token : 1;
        kv_len = a.kv_len[seq];
        token0 = row0 / group;
        token1 = min(n_tokens - 1, (row0 + rows - 1) / group);
        last = min(kv_len - n_tokens + token1, a.width * a.page_size - 1);
        const int low = kv_len - n_tokens + token0 - a.window + 1;
        first = a.window > 0 && low > 0 ? low : 0;
        turns = row0 < n_tokens * group && last >= first ? (last - start()) / kTile4 + 1 : 0;
    }
    __device__ __forceinline__ int start() const { return first & ~15; }
    // Where row `local` of the entry stands in q and out, as token * Hq + head; -1 behind the last.
    __device__ __forceinline__ long row_at(const Attend4& a, int kvh, int local) const {
        const int group = a.Hq / a.Hkv, row = row0 + local, token = row / group;
        return token < n_tokens && first_token + token < a.n_rows ? (long)(first_token + token) * a.Hq + kvh * group + (row - token * group) : -1;
    }
};

// Blocks of an SM, by what registers allow: of float32 or not, with so many groups and rows of a block.
constexpr int blocks_4bit(bool exact, int groups, int rows) {
    const int size = groups * (rows > 8 ? 2 : 1);
    return size >= 6 ? 2 : exact || size > 2 ? 3 : 4;
}
constexpr int kLeastShare4 = 8;         // turns of a block, at least
constexpr int kGap4 = 16;                // turns that a head's start and end are worth
struct Plan4 {
    int share;                          // of a block, in turns
    bool apart;
    __device__ __forceinline__ int gap() const { return apart ? 0 : kGap4; }
    __device__ __forceinline__ int line(int turns) const { return turns == 0 ? 0 : apart ? (turns + share - 1) / share * share : turns + kGap4; }
    // all: turns of all heads; heads: those with turns; most: of one.
    static __device__ __forceinline__ Plan4 of(int all, int heads, int most, int blocks) {
        const int packed = (all + heads * kGap4 + blocks - 1) / blocks;
        int apart = 0x7fffffff;
        if (heads > 0 && heads <= blocks) {
            const int each = blocks / heads;
            apart = (most + each - 1) / each;                                                       // enough blocks for the longest
            if (blocks > heads) apart = min(apart, (all + blocks - heads - 1) / (blocks - heads));  // enough for whatever they are
        }
        const bool is_apart = apart <= packed;
        const int share = max(is_apart ? apart : packed, kLeastShare4);
        return {share, is_apart};
    }
};

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool pred) {
    const int bytes = pred ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}
// D (16x8, f32) += A (16x16, f16, row) * B (16x8, f16, col)
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// (word & MASK) | bits in one instruction: `bits` in a register, of two immediate operands the compiler makes two instructions.
template <uint32_t MASK> __device__ __forceinline__ uint32_t masked_or(uint32_t word, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(word), "n"(MASK), "r"(bits));
    return r;
}
// (128 + c) - 136 = c - 8, exactly.
__device__ __forceinline__ uint32_t centred(uint32_t raw) {
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&raw), __floats2bfloat162_rn(136.0f, 136.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// c - 8 in float16's normal numbers, exactly, of the bits of c and of c << 4.  (float32: the products line subnormal numbers up by the exponent that they
// would have if they were normal, and lose up to ten bits of what they cut off: 1.5e-6 of an output, as it is 3e-7.)
__device__ __forceinline__ uint32_t centred_low(uint32_t bits) {
    const uint32_t raw = bits | 0x64006400u;                    // 1,024 + c
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&raw), __floats2half2_rn(1032.0f, 1032.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t centred_high(uint32_t bits) {
    const uint32_t raw = bits | 0x64006400u;                    // 1,024 + 16 c
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&raw), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <int BYTES> __device__ __forceinline__ void load_shared(uint32_t addr, uint32_t* v) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[4 * i]), "=r"(v[4 * i + 1]), "=r"(v[4 * i + 2]), "=r"(v[4 * i + 3]) : "r"(addr + 16 * i));
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[2 * i]), "=r"(v[2 * i + 1]) : "r"(addr + 8 * i));
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(addr + 4 * i));
    }
}

template <typename T, int G, int NT, int COPIES>
struct Attend4Block {
    static_assert(G % COPIES == 0, "copies take groups in turn");
    static constexpr bool kPairs = COPIES > 1;              // words of two groups as operands
    static constexpr int D = kGroup4 * G, G_ = G, NT_ = NT, COPIES_ = COPIES;
    static constexpr int kColumns = 8 / COPIES;             // rows of the block in 8 columns
    static constexpr int kRows = NT * kColumns;
    static constexpr int GH = G / COPIES;                   // groups of a copy: copy h has h, h + COPIES, ..
    static constexpr int W = kPairs ? G / 2 : G;            // accumulators of 32 channels: of two groups, one for each kind of copy, or of one
    static constexpr bool kExact = sizeof(T) == 4;          // float32: operands of the products in three bfloat16 terms, codes about zero
    static constexpr int kTerms = kExact ? 3 : 1;
    static constexpr float kCodeUp = kExact ? 1.0f : 0x1p24f;           // a code over the operand that stands for it
    // Values keep the offset of their codes, and 136 times the sum of the weights goes through the same products to be taken off every kFold4 turns: the
    // sums are some 16 times as large as the result meanwhile, and the products cut off where float32 rounds (taken off at the end only, outputs
    // of 8,192 keys were 3.0e-3 off, as they are 2.3e-3).  Where there are copies, whose weights share a product.
    static constexpr bool kOffsets = !kExact && COPIES > 1;
    static constexpr int kRow = 16 * G;                     // bytes of a row of codes
    static constexpr int kBuffers = G <= 4 ? 3 : 2;         // a warp's buffers
    static constexpr int kHalfStep = 64 * G, kHalf = 256 * G;            // bytes of 16 keys' steps and codes
    static constexpr int kKeySteps = 2 * kHalf, kValues = kKeySteps + 2 * kHalfStep, kValueSteps = kValues + 2 * kHalf;
    static constexpr int kStage = kValueSteps + 2 * kHalfStep, kRing = kBuffers * kStage;
    static constexpr int kMerge = (kRows * (D + 2) * 4 + 15) / 16 * 16;
    static constexpr int kPerWarp = kRing > kMerge ? kRing : kMerge;
    static constexpr int kQ = kWarps4 * kPerWarp;           // q as the second operand: [term][n][g][lane] of 16 bytes
    static constexpr int kQSums = kTerms * NT * G * 512;    // behind it: [n][g][column] sum, [n][column] factor
    static constexpr int kQLog2 = kQSums + NT * GH * 32, kShared = kQ + kQLog2 + NT * 32;

    // Row k of 16 keys as the products number them stands in row placed(k) of their half of a buffer, and 16-byte chunk c of it at c ^ turned(row): the lanes of
    // either product then read different banks (heads of 128 and 256; the others have some conflicts).
    static __device__ __forceinline__ int placed(int k) { return k ^ ((k >> 1) & 1); }
    static __device__ __forceinline__ int turned(int row) { return G == 4 ? (row >> 1) & 2 : G == 8 ? row & 6 : 0; }

    // The words of a lane's channels 8 t .. + 7 of group g, for a key: t's two 16-bit words side by side.
    static __device__ __forceinline__ uint32_t key_word(const uint32_t (&w)[G], int g) {
        const uint32_t sel = ((g & 1) ? 0x0032u : 0x0010u) | (((G + g) & 1) ? 0x7600u : 0x5400u);
        return __byte_perm(w[g >> 1], w[(G + g) >> 1], sel);
    }
    static __device__ __forceinline__ void load_values(uint32_t rows, int row, int r, uint32_t (&w)[G]) {
        if constexpr (G % 2 == 0) {
            constexpr int kBytes = 2 * G;
            const int chunk = r * kBytes / 16;
            load_shared<kBytes>(rows + row * kRow + (G == 4 || G == 8 ? ((chunk ^ turned(row)) * 16 + r * kBytes % 16) : r * kBytes), w);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint16_t h;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(rows + row * kRow + (r * G + g) * 2));
                w[g] = h;
            }
        }
    }
    // A lane's word of group g of two values, side by side.
    static __device__ __forceinline__ uint32_t value_word(const uint32_t (&lo)[G], const uint32_t (&hi)[G], int g) {
        if constexpr (G % 2 == 0) return __byte_perm(lo[g >> 1], hi[g >> 1], (g & 1) ? 0x7632u : 0x5410u);
        return __byte_perm(lo[g], hi[g], 0x5410u);
    }

    // The sum over a column's copies.
    static __device__ __forceinline__ float over_copies(float v) {
        if (COPIES == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
        if (COPIES >= 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
        return v;
    }

    // State of a warp.  Lane (r, t) = (lane / 4, lane % 4) holds columns 2 t and 2 t + 1 of 8 for each of NT; they belong to copy t COPIES / 4.
    float q_sum[NT][GH][2];                 // sum of a column's q over a group of its copy, over kCodeUp
    float to_log2[NT][2];                   // from a column's sums of products to scores in base 2; above zero (a scale's sign is q's)
    uint32_t bf16_bits;
    uint32_t first_of, second_of;           // byte selections: the first (second) of two weights, where column r's copy wants it, beside zero
    // [w][u]: channels 4 r + 2 u, + 1 (elements 0 1, 2 3) of columns 2 t, 2 t + 1 of group w, or of group 2 w + 1 for odd copies and 2 w for even ones
    float o[NT][W][2][4];
    float least_sum[NT][GH][2];             // this lane's part of sum_j p_j (m_j + 8 s_j)
    float offsets[NT][kOffsets ? GH : 1][4];    // 136 times the sums of the weights of a group of its copy
    float top[NT][2], total[NT][2];
    int pos[NT][2];                         // a column's position

    // The block's q, raw: a lane's channels 8 t .. + 7 of column r in every group of its copy.
    struct RawQ { float v[NT][GH][8]; };
    static __device__ __forceinline__ void read_q(const T* const (&src)[NT], RawQ& raw, int lane) {
        const int t = lane & 3, copy = (lane >> 2) / kColumns;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) raw.v[n][g][e] = 0.0f;
                if (src[n] != nullptr) {
                    load_quad(src[n] + 32 * (copy + COPIES * g) + 8 * t, *reinterpret_cast<float(*)[4]>(raw.v[n][g]));
                    load_quad(src[n] + 32 * (copy + COPIES * g) + 8 * t + 4, *reinterpret_cast<float(*)[4]>(raw.v[n][g] + 4));
                }
            }
    }
    // q as an operand to shared memory, with its sums; the warps share the groups.
    static __device__ __forceinline__ void write_q(RawQ& raw, float scale_log2, uint32_t q_at, int warp, int lane) {
        const int r = lane >> 2, t = lane & 3, copy = r / kColumns;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float most = 0.0f;
#pragma unroll
            for (int g = 0; g < GH; ++g)
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(raw.v[n][g][e]));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            if (COPIES == 4) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
            if (COPIES >= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
            // the row over 2^k, its largest element in [2^14, 2^15): float16 holds 11 bits of all that is above 2^-28 of it
            const int k = min(126, max(-112, (int)(__float_as_uint(most) >> 23) - 127)) - 14;
            const float down = copysignf(__int_as_float((127 - k) << 23), scale_log2);
            if (warp == 0 && t == 0)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(q_at + kQLog2 + (n * 8 + r) * 4), "f"(fmaxf(1.2e-38f, __int_as_float((127 + k) << 23) * kCodeUp * fabsf(scale_log2))) : "memory");      // -inf stays so times it
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                if (g % kWarps4 != warp && GH >= kWarps4) continue;
                if (GH < kWarps4 && g != warp % GH) continue;
                float sum = 0.0f, (&v)[8] = raw.v[n][g];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= down;
                // channels of odd number stand 16 times as high in the codes, unless those are made normal numbers
                constexpr float kDown = kExact ? 1.0f : 0.0625f, kUp = kExact ? 1.0f : 16.0f;
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    uint32_t held[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const __half h = __float2half_rn(v[e] * (e % 2 ? kDown : 1.0f));
                        const float back = __half2float(h) * (e % 2 ? kUp : 1.0f);
                        v[e] -= back;
                        sum += back;
                        held[e] = __half_as_ushort(h);
                    }
                    const uint32_t to = q_at + (term * NT + n) * G * 512 + lane * 16;
                    if constexpr (kPairs) {
                        // words (group pair, half of the channels): four channels each, in the half of the operand that is the copy's
#pragma unroll
                        for (int p = g * COPIES / 2; p < (g + 1) * COPIES / 2; ++p)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t word[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) word[e] = (2 * p + (copy & 1)) % COPIES != copy ? 0u : copy & 1 ? held[4 * i + e] << 16 : held[4 * i + e];
                                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + (2 * p + i) * 512), "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3]) : "memory");
                            }
                    } else {
                        // pairs of channels (e, 4 + e)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to + g * 512), "r"(held[0] | held[4] << 16), "r"(held[1] | held[5] << 16),
                                     "r"(held[2] | held[6] << 16), "r"(held[3] | held[7] << 16) : "memory");
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(q_at + kQSums + ((n * GH + g) * 8 + r) * 4), "f"(sum / kCodeUp) : "memory");
            }
        }
    }
    __device__ __forceinline__ void take_q_sums(uint32_t q_at, int lane) {
        asm volatile("mov.b32 %0, 0x43004300;" : "=r"(bf16_bits));
        const int t = lane & 3;
        if constexpr (kPairs) {
            const bool odd = ((lane >> 2) / kColumns) & 1;
            first_of = odd ? 0x1044u : 0x4410u;
            second_of = odd ? 0x3244u : 0x4432u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(to_log2[n][0]), "=f"(to_log2[n][1]) : "r"(q_at + kQLog2 + (n * 8 + 2 * t) * 4));
#pragma unroll
            for (int g = 0; g < GH; ++g)
                asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(q_sum[n][g][0]), "=f"(q_sum[n][g][1]) : "r"(q_at + kQSums + ((n * GH + g) * 8 + 2 * t) * 4));
        }
    }

    static __device__ __forceinline__ void load_keys(uint32_t half, int row, int t, uint32_t (&w)[G]) {
        if constexpr (G == 4) {
            load_shared<16>(half + row * kRow + ((t ^ turned(row)) * 16), w);
        } else if constexpr (G == 8) {
            load_shared<16>(half + row * kRow + (((2 * t) ^ turned(row)) * 16), w);
            load_shared<16>(half + row * kRow + (((2 * t + 1) ^ turned(row)) * 16), w + 4);
        } else {
            load_shared<4 * G>(half + row * kRow + t * 4 * G, w);
        }
    }

    __device__ __forceinline__ void fold_offsets() {
        if constexpr (kOffsets) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int w = 0; w < W; ++w)
#pragma unroll
                        for (int u = 0; u < 2; ++u) o[n][w][u][c] -= offsets[n][2 * w / COPIES][c];
#pragma unroll
                    for (int j = 0; j < GH; ++j) offsets[n][j][c] = 0.0f;
                }
        }
    }
    // Words of channels 4 r .. + 3 for two columns of the operand: channels 2 u in its rows r, 2 u + 1 in its rows r + 8.
    __device__ __forceinline__ void value_operands(const uint32_t (&z)[2], uint32_t (&a)[2][4]) const {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[u][e] = masked_or<0x000f000fu>(z[e >> 1] >> (8 * u + 4 * (e & 1)), bf16_bits);
                if constexpr (!kOffsets) a[u][e] = centred(a[u][e]);
            }
    }
    // Steps of a key in a copy's groups.
    static __device__ __forceinline__ void load_steps(uint32_t at, int copy, uint32_t (&s)[GH]) {
        if constexpr (kPairs) {
#pragma unroll
            for (int j = 0; j < GH; ++j) load_shared<4>(at + (copy + COPIES * j) * 4, s + j);
        } else {
            load_shared<4 * G>(at, s);
        }
    }

    // The keys from key0 on of which some column does not see some, positions [lowest, highest].  Scores of what a column does not see become -inf.
    // A weight of zero must be nothing whatever the value it belongs to, so steps of values that no column sees, which may be anything, become
    // zero; so do steps that are no numbers of values that only some columns see, and the sums of those columns are none any more.
    template <typename There>
    __device__ __forceinline__ void take_edges(float (&x)[2][NT][4], uint32_t stage, int key0, int lowest, int highest, int window, int lane, There there) {
        const int r = lane >> 2;
        const uint32_t pages = __ballot_sync(0xffffffffu, there(key0 + lane));
        auto sees = [&](int i, int p) { return key0 + i <= p && (window == 0 || key0 + i > p - window) && ((pages >> i) & 1); };
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!sees(16 * half + placed(r) + (e < 2 ? 0 : 8), pos[n][e & 1])) x[half][n][e] = -INFINITY;
        const bool any = key0 + lane <= highest && (window == 0 || key0 + lane > lowest - window) && ((pages >> lane) & 1);
        const bool all = sees(lane, lowest) && sees(lane, highest);
        const uint32_t steps = stage + kValueSteps + lane * 4 * G;
        bool bad = false;
        if (any && !all) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint32_t word;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(word) : "r"(steps + 4 * g));
                bad |= no_number(word);
            }
        }
        if (!any || bad) {
#pragma unroll
            for (int g = 0; g < G; ++g) asm volatile("st.shared.u32 [%0], %1;" ::"r"(steps + 4 * g), "r"(0) : "memory");
        }
        for (uint32_t left = __ballot_sync(0xffffffffu, bad); left != 0; left &= left - 1)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (sees(__ffs(left) - 1, pos[n][c])) total[n][c] = __int_as_float(0x7fc00000);
        __syncwarp();
    }

    // Thirty-two keys.  `edge`: some column does not see some of them; edges(x) then takes those scores away.
    template <typename Edges>
    __device__ __forceinline__ void turn(uint32_t stage, uint32_t q_at, int lane, bool edge, Edges edges) {
        const int r = lane >> 2, t = lane & 3, row0 = placed(r), row1 = row0 + 8, copy = t * COPIES / 4;
        float x[2][NT][4];
        {
            uint32_t w[2][2][G], s[2][2][GH];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    load_keys(stage + half * kHalf, i ? row1 : row0, t, w[half][i]);
                    load_steps(stage + kKeySteps + half * kHalfStep + (i ? row1 : row0) * 4 * G, copy, s[half][i]);
                }
#pragma unroll
            for (int j = 0; j < GH; ++j) {
                float c[2][NT][4];
                // of words or of groups: those whose products belong to slot j of the copies
#pragma unroll
                for (int k = kPairs ? j * COPIES : j; k < (kPairs ? (j + 1) * COPIES : j + 1); ++k) {
                    uint32_t ka[2][2][4];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // words: pair k / 2 of groups, half k % 2 of the channels
                        const uint32_t y[2] = {kPairs ? w[half][0][k / 2 + k % 2 * (G / 2)] : key_word(w[half][0], k), kPairs ? w[half][1][k / 2 + k % 2 * (G / 2)] : key_word(w[half][1], k)};
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                ka[half][i][e] = (i ? y[e & 1] >> 8 : y[e & 1]) & (e < 2 ? 0x000f000fu : 0x00f000f0u);
                                if constexpr (kExact) ka[half][i][e] = e < 2 ? centred_low(ka[half][i][e]) : centred_high(ka[half][i][e]);
                            }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int term = kTerms - 1; term >= 0; --term) {      // the largest terms last
                            uint32_t b[4];
                            load_shared<16>(q_at + ((term * NT + n) * G + k) * 512 + lane * 16, b);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                if (k == (kPairs ? j * COPIES : j) && term == kTerms - 1) mma_f16_first(c[half][n], ka[half][0], b[0], b[1]);
                                else mma_f16(c[half][n], ka[half][0], b[0], b[1]);
                                mma_f16(c[half][n], ka[half][1], b[2], b[3]);
                            }
                        }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = s[half][e >> 1][j];
                        const float step = __uint_as_float(word << 16);
                        float least = __uint_as_float(word & 0xffff0000u);
                        if constexpr (kExact) least = fmaf(8.0f, step, least);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float m = j == 0 ? least * q_sum[n][j][e & 1] : fmaf(least, q_sum[n][j][e & 1], x[half][n][e]);
                            x[half][n][e] = fmaf(step, c[half][n][e], m);
                        }
                    }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[half][n][e] = over_copies(x[half][n][e]);
        if (edge) edges(x);
        bool rises = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // The maximum moves only when a score passes it by more than 2^8: weights stay below 2^8, float32 and bfloat16 have room for them.
#pragma unroll
            for (int c = 0; c < 2; ++c) rises |= fmaxf(fmaxf(x[0][n][c], x[0][n][c + 2]), fmaxf(x[1][n][c], x[1][n][c + 2])) * to_log2[n][c] > top[n][c] + 8.0f;
        }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(fmaxf(x[0][n][c], x[0][n][c + 2]), fmaxf(x[1][n][c], x[1][n][c + 2]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m * to_log2[n][c], top[n][c]);
                    const float shrink = exp2_fast(top[n][c] - m);
                    top[n][c] = m;
                    total[n][c] *= shrink;
#pragma unroll
                    for (int g = 0; g < GH; ++g) {
                        least_sum[n][g][c] *= shrink;
                        if constexpr (kOffsets) {
                            offsets[n][g][c] *= shrink;
                            offsets[n][g][c + 2] *= shrink;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < W; ++w)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            o[n][w][u][c] *= shrink;
                            o[n][w][u][c + 2] *= shrink;
                        }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[half][n][e] = exp2_fast(fmaf(x[half][n][e], to_log2[n][e & 1], -top[n][e & 1]));
#pragma unroll
            for (int c = 0; c < 2; ++c) total[n][c] += (x[0][n][c] + x[0][n][c + 2]) + (x[1][n][c] + x[1][n][c + 2]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t s[2][GH], va[G], vb[G], vc[G], vd[G];
            const uint32_t values = stage + kValues + half * kHalf, steps = stage + kValueSteps + half * kHalfStep;
            load_steps(steps + row0 * 4 * G, copy, s[0]);
            load_steps(steps + row1 * 4 * G, copy, s[1]);
            load_values(values, placed(2 * t), r, va);
            load_values(values, placed(2 * t + 1), r, vb);
            load_values(values, placed(2 * t) + 8, r, vc);
            load_values(values, placed(2 * t + 1) + 8, r, vd);
#pragma unroll
            for (int j = 0; j < GH; ++j) {
                float step[2], middle[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    step[i] = __uint_as_float(s[i][j] << 16);
                    middle[i] = fmaf(8.0f, step[i], __uint_as_float(s[i][j] & 0xffff0000u));
                }
                uint32_t b0[NT][kTerms], b1[NT][kTerms];          // weights of keys 2 t, 2 t + 1, and of those + 8, for column r
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = x[half][n][e] * step[e >> 1];
                        least_sum[n][j][e & 1] = fmaf(x[half][n][e], middle[e >> 1], least_sum[n][j][e & 1]);
                    }
#pragma unroll
                    for (int term = 0; term < kTerms; ++term) {
                        b0[n][term] = transposed_8x8(pack_bf16(w[0], w[1]));
                        b1[n][term] = transposed_8x8(pack_bf16(w[2], w[3]));
                        if constexpr (kExact)
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] -= __bfloat162float(__float2bfloat16_rn(w[e]));
                    }
                    if constexpr (kOffsets) {
                        const uint32_t a[4] = {0x43084308u, 0x43084308u, 0x43084308u, 0x43084308u};
                        mma_bf16(offsets[n][j], a, b0[n][0], b1[n][0]);
                    }
                }
                if constexpr (kPairs) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {                  // keys 2 t and 2 t + 8, then 2 t + 1 and 2 t + 9
                        uint32_t c0[NT][kTerms], c1[NT][kTerms];
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int term = 0; term < kTerms; ++term) {
                                c0[n][term] = __byte_perm(b0[n][term], 0, k ? second_of : first_of);
                                c1[n][term] = __byte_perm(b1[n][term], 0, k ? second_of : first_of);
                            }
#pragma unroll
                        for (int p = j * COPIES / 2; p < (j + 1) * COPIES / 2; ++p) {
                            const uint32_t z[2] = {k ? vb[p] : va[p], k ? vd[p] : vc[p]};
                            uint32_t a[2][4];
                            value_operands(z, a);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int term = kTerms - 1; term >= 0; --term)
#pragma unroll
                                    for (int u = 0; u < 2; ++u) mma_bf16(o[n][p][u], a[u], c0[n][term], c1[n][term]);
                        }
                    }
                } else {
                    const uint32_t z[2] = {value_word(va, vb, j), value_word(vc, vd, j)};
                    uint32_t a[2][4];
                    value_operands(z, a);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int term = kTerms - 1; term >= 0; --term)
#pragma unroll
                            for (int u = 0; u < 2; ++u) mma_bf16(o[n][j][u], a[u], b0[n][term], b1[n][term]);
                }
            }
        }
    }
};

// Which rows of the pools a warp's turns are, and their copies into its buffers.  Turn i of a warp is the keys key0 + i * kWarps4 * kTile4 .. + 31.
// A key that has no page takes row 0 instead, so that no copy depends on anything; `holes` then says that keys have to be looked at one by one.
struct Head4 {
    const int* table;
    int kvh, key0, own, first, last;    // of a warp: its first key and its turns; the first and last key that are seen at all
};
__device__ __forceinline__ int page_of(const Attend4& a, const Head4& head, int key, int& place) {
    const int logical = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
    place = key - logical * a.page_size;
    const int page = head.table[logical];
    page_ok(page, a.bounds);
    return page_or_none(page, a.n_pages);
}

// Pages of whole halves of 16 keys: every half is one run of rows.  A lane keeps the run (row / 16) of half lane % 2 of turn 16 n + lane / 2.
template <typename B>
struct Turns16 {
    uint32_t units, units_next;
    bool holes = false;
    const uint8_t *k, *v, *steps;       // a lane's first chunk of 16 bytes: of codes, and of the steps of one of the pools
    uint32_t code_to, step_to;          // where they go in a buffer

    __device__ __forceinline__ uint32_t load(const Attend4& a, const Head4& head, int turn, int lane) {
        const int key = head.key0 + (turn + (lane >> 1)) * (kWarps4 * kTile4) + (lane & 1) * 16;
        int place, page = 0;
        if (turn + (lane >> 1) < head.own && key <= head.last) page = page_of(a, head, key, place);
        else return 0;
        if (page < 0) holes = true;
        return page < 0 ? 0 : (((uint32_t)page * a.Hkv + head.kvh) * a.page_size + place) / 16;
    }
    __device__ __forceinline__ void begin(const Attend4& a, const Head4& head, int lane) {
        units_next = load(a, head, 0, lane);
        k = a.k.codes + lane * 16;
        v = a.v.codes + lane * 16;
        steps = reinterpret_cast<const uint8_t*>(lane < 16 ? a.k.steps : a.v.steps) + (lane & 15) * 16;
        code_to = lane / B::G_ * B::kRow + ((lane % B::G_ ^ B::turned(lane / B::G_)) * 16);
        step_to = (lane < 16 ? B::kKeySteps : B::kValueSteps) + (lane & 15) * 16;
    }
    // Turn i, in order, into a buffer.
    __device__ __forceinline__ void fill(const Attend4& a, const Head4& head, int i, uint32_t stage, int lane) {
        if ((i & 15) == 0) {
            units = units_next;
            units_next = load(a, head, i + 16, lane);
            holes = __any_sync(0xffffffffu, holes);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t unit = __shfl_sync(0xffffffffu, units, 2 * (i & 15) + half);
            const uint8_t *kc = k + (size_t)unit * B::kHalf, *vc = v + (size_t)unit * B::kHalf, *st = steps + (size_t)unit * B::kHalfStep;
            const uint32_t to = stage + half * B::kHalf;
#pragma unroll
            for (int it = 0; it < (B::G_ + 1) / 2; ++it) {
                if constexpr (B::G_ == 4) {             // eight keys an instruction: the second eight stand 512 bytes behind
                    cp_async16(to + code_to + it * 512, kc + it * 512, true);
                    cp_async16(to + code_to + B::kValues + it * 512, vc + it * 512, true);
                } else {
                    const int j = it * 32 + lane, key = j / B::G_, c = j - key * B::G_;
                    const uint32_t at = to + key * B::kRow + ((c ^ B::turned(key)) * 16);
                    if (B::G_ % 2 == 0 || j < 16 * B::G_) {
                        cp_async16(at, kc + it * 512, true);
                        cp_async16(at + B::kValues, vc + it * 512, true);
                    }
                }
            }
#pragma unroll
            for (int it = 0; it < (4 * B::G_ + 15) / 16; ++it)                   // half the warp a pool
                if (4 * B::G_ % 16 == 0 || it * 16 + (lane & 15) < 4 * B::G_) cp_async16(stage + half * B::kHalfStep + step_to + it * 256, st + it * 256, true);
        }
    }
};

// Pages of any size: key by key.  `row`: of key `lane` of the next turn, `hole`: that key's page is none.  The whole warp has to take a turn's edges or none of
// it, so `holes` is what the warp has voted of the turns that were filled; a lane's own find waits for the fill that needs its row.
template <typename B>
struct TurnsAny {
    uint32_t row;
    bool hole = false, holes = false;

    __device__ __forceinline__ uint32_t load(const Attend4& a, const Head4& head, int turn, int lane) {
        const int key = head.key0 + turn * (kWarps4 * kTile4) + lane;
        int place, page;
        hole = false;
        if (turn >= head.own || key < head.first || key > head.last) return 0;
        page = page_of(a, head, key, place);
        hole = page < 0;
        return page < 0 ? 0 : ((uint32_t)page * a.Hkv + head.kvh) * a.page_size + place;
    }
    __device__ __forceinline__ void begin(const Attend4& a, const Head4& head, int lane) { row = load(a, head, 0, lane); }
    __device__ __forceinline__ void fill(const Attend4& a, const Head4& head, int i, uint32_t stage, int lane) {
        holes = __any_sync(0xffffffffu, hole) || holes;
#pragma unroll
        for (int it = 0; it < B::G_; ++it) {
            const int j = it * 32 + lane, key = j / B::G_, c = j - key * B::G_;
            const size_t at = __shfl_sync(0xffffffffu, row, key);
            const uint32_t to = stage + key * B::kRow + ((c ^ B::turned(key & 15)) * 16);
            cp_async16(to, a.k.codes + at * B::kRow + c * 16, true);
            cp_async16(to + B::kValues, a.v.codes + at * B::kRow + c * 16, true);
            cp_async4(stage + B::kKeySteps + j * 4, reinterpret_cast<const uint32_t*>(a.k.steps) + at * B::G_ + c, true);
            cp_async4(stage + B::kValueSteps + j * 4, reinterpret_cast<const uint32_t*>(a.v.steps) + at * B::G_ + c, true);
        }
        row = load(a, head, i + 1, lane);
    }
};

// Where a block's run of the line begins: every block looks at all entries; block 0 leaves the plan for the kernel that joins.
struct Run4 {
    int from, to, entry, offset;        // [from, to) of the line, the first of them `offset` into `entry`
    Plan4 plan;
};
__device__ __forceinline__ Run4 run_of(const Attend4& a, int rows) {
    __shared__ int sums[3][kWarps4], found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, entries = a.n_seqs * a.row_blocks;
    int all = 0, heads = 0, most = 0, mine = 0;
    for (int e = threadIdx.x; e < entries; e += kWarps4 * 32) {
        const int n = Entry4(a, e, rows).turns;
        if (e < kWarps4 * 32) mine = n;
        all += n;
        heads += n > 0;
        most = max(most, n);
    }
    all = __reduce_add_sync(0xffffffffu, all);
    heads = __reduce_add_sync(0xffffffffu, heads);
    most = __reduce_max_sync(0xffffffffu, most);
    if (entries > 32) {                 // else the first warp has seen them all
        if (lane == 0) { sums[0][warp] = all; sums[1][warp] = heads; sums[2][warp] = most; }
        __syncthreads();
        all = heads = most = 0;
#pragma unroll
        for (int w = 0; w < kWarps4; ++w) { all += sums[0][w]; heads += sums[1][w]; most = max(most, sums[2][w]); }
    } else {
        if (threadIdx.x == 0) { sums[0][0] = all; sums[1][0] = heads; sums[2][0] = most; }
        __syncthreads();
        all = sums[0][0]; heads = sums[1][0]; most = sums[2][0];
    }
    Run4 run;
    run.plan = Plan4::of(all * a.Hkv, heads * a.Hkv, most, a.blocks);
    run.from = (int)min(0x7fffffffLL, (long long)blockIdx.x * run.plan.share);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = run.plan.apart ? -run.plan.share : run.plan.share;
    int before = 0;
    for (int e0 = 0; e0 < entries; e0 += kWarps4 * 32) {
        const int e = e0 + threadIdx.x;
        const int n = run.plan.line(e0 == 0 ? mine : e < entries ? Entry4(a, e, rows).turns : 0) * a.Hkv;
        int upto = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += v;
        }
        __syncthreads();                // `sums` have been read
        if (lane == 31) sums[0][warp] = upto;
        __syncthreads();
        int here = before - n + upto;
#pragma unroll
        for (int w = 0; w < kWarps4; ++w) {
            if (w < warp) here += sums[0][w];
            before += sums[0][w];
        }
        if (blockIdx.x == 0 && e < entries) a.plan[1 + e] = here;
        if (run.from >= here && run.from < here + n) {
            found[0] = e;
            found[1] = run.from - here;
        }
        if (blockIdx.x != 0 && before > run.from) break;
    }
    __syncthreads();
    // the line's length is known where it was gone through to the end; who begins before it ends has been found
    run.to = run.from < before ? run.from + run.plan.share : run.from;
    run.entry = found[0];
    run.offset = found[1];
    return run;
}

// Turns [skipped, skipped + n_turns) of a head by the warps of a block.  Afterwards every warp's sums stand in its shared memory: [row][D], then
// (maximum, sum of weights) of each row; block_sum adds them up.
template <typename T, typename B, typename Turns>
__device__ __forceinline__ void attend_part(const Attend4& a, const Entry4& entry, int kvh, int skipped, int n_turns, uint8_t* shared) {
    constexpr int D = B::D, NT = B::NT_, COPIES = B::COPIES_;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(shared) + warp * B::kPerWarp, q_at = smem_u32(shared) + B::kQ;
    const int own = n_turns > warp ? (n_turns - warp + kWarps4 - 1) / kWarps4 : 0;
    const Head4 head = {a.table + (size_t)entry.seq * a.width, kvh, entry.start() + (skipped + warp) * kTile4, own, entry.first, entry.last};
    Turns turns;
    turns.begin(a, head, lane);
    const T* src[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const long at = entry.row_at(a, kvh, B::kColumns * n + r % B::kColumns);
        src[n] = at < 0 ? nullptr : reinterpret_cast<const T*>(a.q) + at * D;
    }
    typename B::RawQ raw;
    B::read_q(src, raw, lane);
#pragma unroll
    for (int i = 0; i < B::kBuffers - 1; ++i) {
        if (i < own) turns.fill(a, head, i, ring + i * B::kStage, lane);
        cp_async_commit();
    }
    B::write_q(raw, a.scale_log2, q_at, warp, lane);

    B b;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int group = a.Hq / a.Hkv;
            b.pos[n][c] = min(entry.last, entry.kv_len - entry.n_tokens + min(entry.n_tokens - 1, (entry.row0 + B::kColumns * n + (2 * t + c) % B::kColumns) / group));
            b.top[n][c] = kLowest4;
            b.total[n][c] = 0.0f;
#pragma unroll
            for (int g = 0; g < B::GH; ++g) {
                b.least_sum[n][g][c] = 0.0f;
                if (B::kOffsets) b.offsets[n][g][c] = b.offsets[n][g][c + 2] = 0.0f;
            }
#pragma unroll
            for (int w = 0; w < B::W; ++w)
#pragma unroll
                for (int u = 0; u < 2; ++u) b.o[n][w][u][c] = b.o[n][w][u][c + 2] = 0.0f;
        }
    // turns [inner_from, inner_to) are seen whole by every column
    const int before = entry.kv_len - entry.n_tokens;
    const int lowest = min(entry.last, before + entry.token0), highest = min(entry.last, before + entry.token1);
    const int above = a.window > 0 ? before + entry.token1 - a.window - head.key0 + 1 : 0;
    const int inner_from = above > 0 ? (above + kWarps4 * kTile4 - 1) / (kWarps4 * kTile4) : 0;
    const int inner_to = lowest - head.key0 >= kTile4 - 1 ? (lowest - head.key0 - (kTile4 - 1)) / (kWarps4 * kTile4) + 1 : 0;
    __syncthreads();
    b.take_q_sums(q_at, lane);

    uint32_t stage = ring, free = ring + (B::kBuffers - 1) * B::kStage;
    for (int i = 0; i < own; ++i) {
        cp_async_wait<B::kBuffers - 2>();
        __syncwarp();
        if (i + B::kBuffers - 1 < own) turns.fill(a, head, i + B::kBuffers - 1, free, lane);
        cp_async_commit();
        b.turn(stage, q_at, lane, i < inner_from || i >= inner_to || turns.holes, [&](auto& x) {
            b.take_edges(x, stage, head.key0 + i * (kWarps4 * kTile4), lowest, highest, a.window, lane, [&](int key) {
                int place;
                return !turns.holes || (key >= head.first && key <= head.last && page_of(a, head, key, place) >= 0);
            });
        });
        if ((i & (kFold4 - 1)) == kFold4 - 1) b.fold_offsets();
        free = stage;
        stage = stage == ring + (B::kBuffers - 1) * B::kStage ? ring : stage + B::kStage;
        __syncwarp();
    }
    b.fold_offsets();
    cp_async_wait<0>();
    __syncwarp();
    // The warp's sums to its own shared memory (the ring is done with): [column][D], then maxima and totals.
    float* mine = reinterpret_cast<float*>(shared + warp * B::kPerWarp);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int column = B::kColumns * n + (2 * t + c) % B::kColumns, copy = t * COPIES / 4;
            float total = b.total[n][c];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
            float least[B::GH];
#pragma unroll
            for (int j = 0; j < B::GH; ++j) {
                least[j] = b.least_sum[n][j][c];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) least[j] += __shfl_xor_sync(0xffffffffu, least[j], off);
            }
#pragma unroll
            for (int w = 0; w < B::W; ++w) {
                const int g = B::kPairs ? 2 * w + (copy & 1) : w;
                const float m = least[B::kPairs ? 2 * w / COPIES : w];
                if (!B::kPairs || g % COPIES == copy)
                    *reinterpret_cast<float4*>(mine + column * D + 32 * g + 4 * r) =
                        make_float4(b.o[n][w][0][c] + m, b.o[n][w][0][c + 2] + m, b.o[n][w][1][c] + m, b.o[n][w][1][c + 2] + m);
            }
            if (r == 0 && copy == 0) {
                mine[B::kRows * D + 2 * column] = b.top[n][c];
                mine[B::kRows * D + 2 * column + 1] = total;
            }
        }
    __syncthreads();
}
// Four channels of a row, the warps' parts together: not divided by the sum of weights.
template <typename B>
__device__ __forceinline__ void block_sum(const uint8_t* shared, int column, int quad, float& top, float& total, float (&v)[4]) {
    constexpr int D = B::D;
    float tops[kWarps4];
    top = kLowest4;
    total = v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps4; ++w) {
        tops[w] = reinterpret_cast<const float*>(shared + w * B::kPerWarp)[B::kRows * D + 2 * column];
        top = fmaxf(top, tops[w]);
    }
#pragma unroll
    for (int w = 0; w < kWarps4; ++w) {
        const float* theirs = reinterpret_cast<const float*>(shared + w * B::kPerWarp);
        const float f = exp2_fast(tops[w] - top);
        const float4 s = *reinterpret_cast<const float4*>(theirs + column * D + 4 * quad);
        total += f * theirs[B::kRows * D + 2 * column + 1];
        v[0] += f * s.x; v[1] += f * s.y; v[2] += f * s.z; v[3] += f * s.w;
    }
}
template <typename T> __device__ __forceinline__ void store_weighed(T* out, float total, float (&v)[4]) {
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = total == 0.0f ? 0.0f : v[e] * inverse;
    store_quad(out, v);
}

template <typename T, int G, int NT, int COPIES, typename Turns, int BLOCKS>
__global__ void __launch_bounds__(kWarps4 * 32, BLOCKS) attend_4bit_kernel(const Attend4 a) {
    using B = Attend4Block<T, G, NT, COPIES>;
    constexpr int D = B::D;
    pdl_wait();
    extern __shared__ __align__(128) uint8_t shared[];
    const int lane = threadIdx.x & 31;
    pdl_trigger();                      // all blocks are here at once: what joins may come as they end
    Run4 run = run_of(a, B::kRows);
    while (run.from < run.to) {
        const Entry4 entry(a, run.entry, B::kRows);
        const int line = run.plan.line(entry.turns);
        if (run.offset >= line * a.Hkv) {                // on to the next entry that has turns, 32 looked at together
            const int entries = a.n_seqs * a.row_blocks;
            uint32_t some = 0;
            for (++run.entry; run.entry < entries && some == 0; run.entry += 32)
                some = __ballot_sync(0xffffffffu, run.entry + lane < entries && Entry4(a, min(run.entry + lane, entries - 1), B::kRows).turns > 0);
            if (some == 0) break;
            run.entry += __ffs(some) - 33;
            run.offset = 0;
            continue;
        }
        // the part [skipped, skipped + n_turns) of a head
        const int kvh = run.offset / line, at_line = run.offset - kvh * line, taken = min(line - at_line, run.to - run.from);
        const int skipped = max(0, at_line - run.plan.gap()), n_turns = min(entry.turns, at_line + taken - run.plan.gap()) - skipped;
        run.from += taken;
        run.offset += taken;
        if (n_turns <= 0) continue;
        attend_part<T, B, Turns>(a, entry, kvh, skipped, n_turns, shared);
        const bool whole = n_turns == entry.turns;
        const int place = 2 * blockIdx.x + (skipped > 0 ? 0 : 1);        // a head that another block began, or one that another ends
        for (int i = threadIdx.x; i < B::kRows * (D / 4); i += kWarps4 * 32) {
            const int column = i / (D / 4), quad = i - column * (D / 4);
            const long at = entry.row_at(a, kvh, column);
            if (at < 0) continue;
            float top, total, v[4];
            block_sum<B>(shared, column, quad, top, total, v);
            if (whole) {
                store_weighed(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, total, v);
            } else {
                store_quad(a.sums + ((size_t)place * B::kRows + column) * D + 4 * quad, v);
                if (quad == 0) *reinterpret_cast<float2*>(a.sums + (size_t)2 * a.blocks * B::kRows * D + ((size_t)place * B::kRows + column) * 2) = make_float2(top, total);
            }
        }
        __syncthreads();
    }
}

// A head a cluster (of one block: a block): its parts are joined through the blocks' shared memory, and nothing needs to be known of the others.
template <typename T, int G, int NT, int COPIES, typename Turns, int BLOCKS>
__global__ void __launch_bounds__(kWarps4 * 32, BLOCKS) attend_4bit_cluster_kernel(const Attend4 a) {
    namespace cg = cooperative_groups;
    using B = Attend4Block<T, G, NT, COPIES>;
    constexpr int D = B::D;
    pdl_wait();
    extern __shared__ __align__(128) uint8_t shared[];
    const int parts = gridDim.x, part = blockIdx.x, kvh = blockIdx.y / a.row_blocks;
    const Entry4 entry(a, blockIdx.z * a.row_blocks + blockIdx.y - kvh * a.row_blocks, B::kRows);
    if (entry.row0 >= entry.n_tokens * (a.Hq / a.Hkv)) return;                   // the whole cluster
    const int share = (entry.turns + parts - 1) / parts, skipped = part * share;
    attend_part<T, B, Turns>(a, entry, kvh, skipped, max(0, min(share, entry.turns - skipped)), shared);
    pdl_trigger();
    float* mine = reinterpret_cast<float*>(shared + B::kShared);                 // [row][D], then (maximum, sum of weights) of each
    for (int i = threadIdx.x; i < B::kRows * (D / 4); i += kWarps4 * 32) {
        const int column = i / (D / 4), quad = i - column * (D / 4);
        float top, total, v[4];
        block_sum<B>(shared, column, quad, top, total, v);
        if (parts == 1) {
            const long at = entry.row_at(a, kvh, column);
            if (at >= 0) store_weighed(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, total, v);
        } else {
            *reinterpret_cast<float4*>(mine + column * D + 4 * quad) = make_float4(v[0], v[1], v[2], v[3]);
            if (quad == 0) *reinterpret_cast<float2*>(mine + B::kRows * D + 2 * column) = make_float2(top, total);
        }
    }
    if (parts == 1) return;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = part * kWarps4 * 32 + threadIdx.x; i < B::kRows * (D / 4); i += parts * kWarps4 * 32) {
        const int column = i / (D / 4), quad = i - column * (D / 4);
        const long at = entry.row_at(a, kvh, column);
        if (at < 0) continue;
        float2 ml[8];
        float4 s[8];
        float top = kLowest4, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < parts) {
                const float* theirs = cluster.map_shared_rank(mine, p);
                ml[p] = *reinterpret_cast<const float2*>(theirs + B::kRows * D + 2 * column);
                s[p] = *reinterpret_cast<const float4*>(theirs + column * D + 4 * quad);
                top = fmaxf(top, ml[p].x);
            }
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < parts) {
                const float f = exp2_fast(ml[p].x - top);
                total += f * ml[p].y;
                v[0] += f * s[p].x; v[1] += f * s[p].y; v[2] += f * s[p].z; v[3] += f * s[p].w;
            }
        store_weighed(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, total, v);
    }
    cluster.sync();                     // nobody leaves while its shared memory is read
}

// The rows of heads that several blocks had, joined; zeros where there is no key.  A block a row and head, its warps every fourth part.
template <typename T>
__global__ void __launch_bounds__(128) join_4bit_kernel(const Attend4 a, int D, int rows) {
    pdl_wait();
    __shared__ float shared[4][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.Hq / a.Hkv, seq = blockIdx.y;
    const int token = blockIdx.x / a.Hq, head = blockIdx.x - token * a.Hq, kvh = head / group, row = token * group + head - kvh * group;
    const Entry4 entry(a, seq * a.row_blocks + row / rows, rows);
    const long at = token < entry.n_tokens ? entry.row_at(a, kvh, row % rows) : -1;
    if (at < 0) return;
    float v[2][4] = {};
    if (entry.turns > 0) {
        const Plan4 plan = {abs(a.plan[0]), a.plan[0] < 0};
        const int from = a.plan[1 + seq * a.row_blocks + row / rows] + kvh * plan.line(entry.turns) + plan.gap();
        const int block0 = from / plan.share, parts = (from + entry.turns - 1) / plan.share - block0 + 1;
        if (parts == 1) return;                          // its block has written it
        const float* ml = a.sums + (size_t)2 * a.blocks * rows * D;
        // part p is block0 + p's: the first of them began the head, unless the head's first turn is the first of the block
        auto place = [&](int p) { return (size_t)(2 * (block0 + p) + (p > 0 ? 0 : 1)) * rows + row % rows; };
        float top = kLowest4, total = 0.0f;
        for (int p = lane; p < parts; p += 32) top = fmaxf(top, ml[2 * place(p)]);
        top = warp_max(top);
        for (int p = lane; p < parts; p += 32) total += exp2_fast(ml[2 * place(p)] - top) * ml[2 * place(p) + 1];
        total = warp_sum(total);
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll 4
        for (int p = warp; p < parts; p += 4) {
            const float f = exp2_fast(ml[2 * place(p)] - top);
            const float* s = a.sums + place(p) * D;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (4 * (lane + 32 * j) < D) {
                    float w[4];
                    load_quad(s + 4 * (lane + 32 * j), w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] = fmaf(f, w[e], v[j][e]);
                }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (4 * (lane + 32 * j) < D) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = total == 0.0f ? 0.0f : v[j][e] * inverse;
                *reinterpret_cast<float4*>(shared[warp] + 4 * (lane + 32 * j)) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
            }
        __syncthreads();
    } else if (warp == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (4 * (lane + 32 * j) < D) store_quad(reinterpret_cast<T*>(a.out) + at * D + 4 * (lane + 32 * j), v[j]);
        return;
    } else {
        return;
    }
    const int quad = threadIdx.x;
    if (4 * quad < D) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (shared[0][4 * quad + e] + shared[1][4 * quad + e]) + (shared[2][4 * quad + e] + shared[3][4 * quad + e]);
        store_quad(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, w);
    }
}

// Behind a dense kernel over expanded pages, where pages that are none stand as keys of zeros: the rows of sequences that see such, once more on codes.
// A row of blocks a sequence; all others' have nothing to do but to look at the table, which they do while the dense kernel runs: that one was launched
// behind everything that writes tables and lengths.  (us without such pages, without this launch and with it, of two runs: 512 tokens over 6,000 keys
// 63.0, 64.2 and 64.0, 65.7; 2,048 tokens 150.9, 151.7 and 151.2, 152.2.  All behind pdl_wait 62.6, 65.5.)
template <typename T, int G, int NT, typename Turns, int BLOCKS>
__global__ void __launch_bounds__(kWarps4 * 32, BLOCKS) attend_4bit_holes_kernel(const Attend4 a) {
    using B = Attend4Block<T, G, NT, 1>;
    constexpr int D = B::D;
    extern __shared__ __align__(128) uint8_t shared[];
    const int seq = blockIdx.y, n_tokens = a.cu_q[seq + 1] - a.cu_q[seq], kv_len = a.kv_len[seq];
    const int low = kv_len - n_tokens - a.window + 1, first = a.window > 0 && low > 0 ? low : 0, last = min(kv_len, a.width * a.page_size) - 1;
    bool hole = false;
    if (n_tokens > 0 && last >= first)
        for (int page = first / a.page_size + threadIdx.x; page <= last / a.page_size; page += kWarps4 * 32)
            hole |= page_or_none(a.table[(size_t)seq * a.width + page], a.n_pages) < 0;
    hole = __syncthreads_or(hole);
    pdl_trigger();
    pdl_wait();                         // the dense kernel has written its rows
    if (!hole) return;
    for (int item = blockIdx.x; item < a.Hkv * a.row_blocks; item += gridDim.x) {
        const int kvh = item / a.row_blocks;
        const Entry4 entry(a, seq, item - kvh * a.row_blocks, B::kRows);
        if (entry.row0 >= n_tokens * (a.Hq / a.Hkv)) continue;
        attend_part<T, B, Turns>(a, entry, kvh, 0, entry.turns, shared);
        for (int i = threadIdx.x; i < B::kRows * (D / 4); i += kWarps4 * 32) {
            const int column = i / (D / 4), quad = i - column * (D / 4);
            const long at = entry.row_at(a, kvh, column);
            if (at < 0) continue;
            float top, total, v[4];
            block_sum<B>(shared, column, quad, top, total, v);
            store_weighed(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, total, v);
        }
        __syncthreads();
    }
}
template <typename T, int G, int NT, template <typename> class Turns>
int launch_attend_4bit_holes(const Attend4& a, int sms, cudaStream_t stream) {
    using B = Attend4Block<T, G, NT, 1>;
    constexpr int kBlocks = blocks_4bit(sizeof(T) == 4, G, B::kRows);
    auto kernel = attend_4bit_holes_kernel<T, G, NT, Turns<B>, kBlocks>;
    static SmemLimit limit;
    if (const int rc = limit.allow(kernel, B::kShared)) return rc;
    const long long items = (long long)a.Hkv * a.row_blocks, each = sms / a.n_seqs;           // a block an SM
    return launch_pdl(kernel, dim3((unsigned)(items < each ? items : each > 0 ? each : 1), a.n_seqs), dim3(kWarps4 * 32), B::kShared, stream, a);
}

template <typename T, int G, int NT, int COPIES, template <typename> class Turns>
int launch_attend_4bit(const Attend4& a, int most_tokens, cudaStream_t stream) {
    using B = Attend4Block<T, G, NT, COPIES>;
    constexpr int kBlocks = blocks_4bit(sizeof(T) == 4, G, B::kRows);
    auto kernel = attend_4bit_kernel<T, G, NT, COPIES, Turns<B>, kBlocks>;
    if (a.blocks < 0) {                 // clusters of -blocks
        auto clusters = attend_4bit_cluster_kernel<T, G, NT, COPIES, Turns<B>, kBlocks>;
        constexpr int kBytes = B::kShared + B::kRows * (B::D + 2) * 4;
        static SmemLimit limit;
        if (const int rc = limit.allow(clusters, kBytes)) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(-a.blocks, a.Hkv * a.row_blocks, a.n_seqs);
        cfg.blockDim = dim3(kWarps4 * 32);
        cfg.dynamicSmemBytes = kBytes;
        cfg.stream = stream;
        cudaLaunchAttribute attrs[2];
        attrs[0].id = cudaLaunchAttributeClusterDimension;
        attrs[0].val.clusterDim.x = -a.blocks;
        attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
        attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attrs;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        return (int)cudaLaunchKernelEx(&cfg, clusters, a);
    }
    static SmemLimit limit;
    if (const int rc = limit.allow(kernel, B::kShared)) return rc;
    if (const int rc = launch_pdl(kernel, dim3(a.blocks), dim3(kWarps4 * 32), B::kShared, stream, a)) return rc;
    return launch_pdl(join_4bit_kernel<T>, dim3(most_tokens * a.Hq, a.n_seqs), dim3(128), 0, stream, a, B::D, B::kRows);
}

template <typename T, int G, template <typename> class Turns>
int launch_attend_4bit_of(const Attend4& a, int rows, int most_tokens, cudaStream_t stream) {
    if constexpr (G % 4 == 0)
        if (rows == 2) return launch_attend_4bit<T, G, 1, 4, Turns>(a, most_tokens, stream);
    if constexpr (G % 2 == 0)
        if (rows == 4) return launch_attend_4bit<T, G, 1, 2, Turns>(a, most_tokens, stream);
    if constexpr (sizeof(T) == 2 && G <= 4)
        if (rows == 16) return launch_attend_4bit<T, G, 2, 1, Turns>(a, most_tokens, stream);
    return rows == 8 ? launch_attend_4bit<T, G, 1, 1, Turns>(a, most_tokens, stream) : PB_ERR_BAD_SIZE;
}

template <typename T, int G>
int launch_attend_4bit_of(const Attend4& a, int rows, int most_tokens, cudaStream_t stream) {
    return a.page_size % 16 == 0 ? launch_attend_4bit_of<T, G, Turns16>(a, rows, most_tokens, stream) : launch_attend_4bit_of<T, G, TurnsAny>(a, rows, most_tokens, stream);
}

template <typename T>
int launch_attend_4bit_of(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream) {
    switch (groups) {
        case 1: return launch_attend_4bit_of<T, 1>(a, rows, most_tokens, stream);
        case 2: return launch_attend_4bit_of<T, 2>(a, rows, most_tokens, stream);
        case 3: return launch_attend_4bit_of<T, 3>(a, rows, most_tokens, stream);
        case 4: return launch_attend_4bit_of<T, 4>(a, rows, most_tokens, stream);
        case 5: return launch_attend_4bit_of<T, 5>(a, rows, most_tokens, stream);
        case 6: return launch_attend_4bit_of<T, 6>(a, rows, most_tokens, stream);
        case 7: return launch_attend_4bit_of<T, 7>(a, rows, most_tokens, stream);
        case 8: return launch_attend_4bit_of<T, 8>(a, rows, most_tokens, stream);
    }
    return PB_ERR_BAD_SIZE;
}

int attend_4bit_f32(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream);      // rows of a block: attention_4bit_rows
int attend_4bit_bf16(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream);

}  // namespace pb
