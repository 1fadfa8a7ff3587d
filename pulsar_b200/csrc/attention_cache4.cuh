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
// A code becomes an operand by one logical instruction for two of them: 128 + c is the bits 0x4300 | c in bfloat16, 1,024 + c is 0x6400 | c in
// float16 and 1,024 + 16 c is 0x6400 | c << 4, which spares a shift: keys are taken in float16, with q scaled to it by a power of two a row.
// Values stay in bfloat16, whose range a weight times a step needs.  A block takes one sequence, kv head,
// up to 8 NT rows (query heads of the kv head, tokens) and a part of the keys; its warps take runs of 16 keys in turn, each through a
// ring of its own in shared memory, so that nobody waits for anybody until the end.  mma.sync m16n8k16 has the keys in its 16 rows for
// the scores and the channels for the weighted sum, and the rows of the block in its 8 columns, where rows in its 16 would be mostly empty.
// A block of 4 rows (2) stands in the columns twice (four times): the products of half (a quarter) of the groups go to each copy, so that no lane
// computes for an empty column what belongs to a key and column: offsets, steps and least values, weights.  The weights change places
// between the two products by movmatrix.
// (tcgen05 would want codes as bfloat16 in shared memory, which is more traffic there than all the rest; what bounds this kernel are instructions
// on codes and bytes, not products.)
#pragma once

#include <cuda_fp16.h>

#include "cache4.cuh"
#include "mma_common.cuh"

namespace pb {

constexpr int kTile4 = 16;              // keys of a warp's turn
constexpr int kWarps4 = 4;
constexpr int kStages4 = 4;             // turns in a warp's ring
constexpr uint32_t kNoRow = 0xffffffffu;
constexpr float kLowest4 = -3.0e38f;    // a running maximum before the first key

struct Attend4 {
    const void* q;
    void* out;
    Pool4 k, v;
    float* sums;                        // [rows of q, Hq, parts, D] and behind it [.., 2] (maximum, sum of weights); with more than one part
    const int* table;
    const int* kv_len;
    const int* cu_q;                    // null: one token each
    int width, n_rows, n_seqs, Hq, Hkv, page_size, page_shift, n_pages, parts, part_keys, row_blocks, window;
    float scale_log2;
    PoolBounds bounds;
};

// The keys [first, last] that any of the block's rows sees, and where the part lies in them.
struct Span4 {
    int first, last;
    __device__ __forceinline__ Span4(const Attend4& a, int kv_len, int n_tokens, int token0, int token1) {
        last = min(kv_len - n_tokens + token1, a.width * a.page_size - 1);
        const int low = kv_len - n_tokens + token0 - a.window + 1;
        first = a.window > 0 && low > 0 ? low : 0;
    }
    __device__ __forceinline__ int start() const { return first & ~(kTile4 - 1); }
    __device__ __forceinline__ int parts(const Attend4& a) const { return last < first ? 0 : min(a.parts, (last - start()) / a.part_keys + 1); }
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
// The same of float16's 1,024 + c and 1,024 + 16 c.
__device__ __forceinline__ uint32_t centred_low(uint32_t raw) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&raw), __floats2half2_rn(1032.0f, 1032.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t centred_high(uint32_t raw) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&raw), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
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
    static_assert(G % COPIES == 0 && (NT == 1 || COPIES == 1), "copies of single columns' groups");
    static constexpr int D = kGroup4 * G, G_ = G;
    static constexpr int kColumns = 8 / COPIES;             // rows of the block in 8 columns
    static constexpr int kRows = NT * kColumns;
    static constexpr int GH = G / COPIES;                   // groups of a copy: copy h has h GH ..
    static constexpr bool kExact = sizeof(T) == 4;          // float32: operands of the products in three bfloat16 terms, codes about zero
    static constexpr int kTerms = kExact ? 3 : 1;
    static constexpr int kRow = 16 * G;                     // bytes of a row of codes
    static constexpr int kKeySteps = kTile4 * kRow, kValues = kKeySteps + kTile4 * 4 * G, kValueSteps = kValues + kTile4 * kRow;
    static constexpr int kSeen = kValueSteps + kTile4 * 4 * G, kStage = kSeen + 16;
    static constexpr int kRing = kStages4 * kStage;
    static constexpr int kMerge = (kRows * (D + 2) * 4 + 15) / 16 * 16;
    static constexpr int kPerWarp = kRing > kMerge ? kRing : kMerge;
    static constexpr int kShared = kWarps4 * kPerWarp;

    // Row k of 16 keys as the products number them stands in row placed(k) of a stage, and 16-byte chunk c of it at c ^ turned(row): the lanes of
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
    uint32_t qb[kTerms][NT][G][2][2];       // q as the second operand: column r, channels 32 g + 8 t + ..
    float q_sum[NT][GH][2];                 // sum of a column's q over a group of its copy
    float q_offset[NT][GH][2];              // what the offsets of the codes add to a column's products
    float to_log2[NT][2];                   // from a column's sums of products to scores in base 2
    uint32_t f16_bits, bf16_bits;
    float o[NT][G][2][4];                   // [u]: channels 32 g + 4 r + 2 u, + 1 (elements 0 1, 2 3) of columns 2 t, 2 t + 1; of the columns' copies that have g
    float least_sum[NT][GH][2];             // this lane's part of sum_j p_j (m_j + 8 s_j)
    float top[NT][2], total[NT][2];
    int pos[NT][2];                         // a column's position

    __device__ __forceinline__ void load_q(const T* const (&src)[NT], float scale_log2, int lane) {
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(f16_bits));
        asm volatile("mov.b32 %0, 0x43004300;" : "=r"(bf16_bits));
        const int t = lane & 3, copy = (lane >> 2) / kColumns;             // of column r
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float v[GH][8], most = 0.0f;
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[g][e] = 0.0f;
                if (src[n] != nullptr) {
                    load_quad(src[n] + 32 * (copy * GH + g) + 8 * t, *reinterpret_cast<float(*)[4]>(v[g]));
                    load_quad(src[n] + 32 * (copy * GH + g) + 8 * t + 4, *reinterpret_cast<float(*)[4]>(v[g] + 4));
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[g][e]));
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            if (COPIES == 4) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
            if (COPIES >= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
            // the row over 2^k, its largest element in [1, 2); float16 then rounds what is below 2^-14 to 2^-25 of that
            const int k = most > 0.0f ? min(126, max(-126, ilogbf(most))) : 0;
            const float down = __int_as_float((127 - k) << 23), up = __int_as_float((127 + k) << 23) * scale_log2;
            to_log2[n][0] = __shfl_sync(0xffffffffu, up, 8 * t);
            to_log2[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                float sum = 0.0f, offset = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[g][e] *= down;
                    sum += v[g][e];
                }
                // words: pairs of channels (e, 4 + e); those of odd e stand 16 times as high in the codes
                constexpr float kHigh = kExact ? 1.0f : 0.0625f;
#pragma unroll
                for (int term = 0; term < kTerms; ++term)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float lo = __half2float(__float2half_rn(v[g][e])), hi = __half2float(__float2half_rn(v[g][4 + e])), by = e % 2 ? kHigh : 1.0f;
                        const uint32_t both = pack_f16(lo * by, hi * by);
#pragma unroll
                        for (int h = 0; h < COPIES; ++h) qb[term][n][h * GH + g][e >> 1][e & 1] = copy == h ? both : 0u;
                        if constexpr (kExact) {
                            v[g][e] -= lo;
                            v[g][4 + e] -= hi;
                        } else {
                            const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&both));
                            offset += 1024.0f * (held.x + held.y);
                        }
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                offset += __shfl_xor_sync(0xffffffffu, offset, 1);
                offset += __shfl_xor_sync(0xffffffffu, offset, 2);
                q_sum[n][g][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                q_sum[n][g][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                q_offset[n][g][0] = __shfl_sync(0xffffffffu, offset, 8 * t);
                q_offset[n][g][1] = __shfl_sync(0xffffffffu, offset, 8 * t + 4);
            }
        }
    }

    // Sixteen keys.  EDGE: some column does not see some of them.
    template <bool EDGE>
    __device__ __forceinline__ void turn(uint32_t stage, int key0, uint32_t seen, int window, int lane) {
        const int r = lane >> 2, t = lane & 3, row0 = placed(r), row1 = row0 + 8, copy = t * COPIES / 4;
        float x[NT][4];
        {
            uint32_t w0[G], w1[G], s0[GH], s1[GH];
            if constexpr (G == 4) {
                load_shared<16>(stage + row0 * kRow + ((t ^ turned(row0)) * 16), w0);
                load_shared<16>(stage + row1 * kRow + ((t ^ turned(row1)) * 16), w1);
            } else if constexpr (G == 8) {
                load_shared<16>(stage + row0 * kRow + (((2 * t) ^ turned(row0)) * 16), w0);
                load_shared<16>(stage + row0 * kRow + (((2 * t + 1) ^ turned(row0)) * 16), w0 + 4);
                load_shared<16>(stage + row1 * kRow + (((2 * t) ^ turned(row1)) * 16), w1);
                load_shared<16>(stage + row1 * kRow + (((2 * t + 1) ^ turned(row1)) * 16), w1 + 4);
            } else {
                load_shared<4 * G>(stage + row0 * kRow + t * 4 * G, w0);
                load_shared<4 * G>(stage + row1 * kRow + t * 4 * G, w1);
            }
            load_shared<4 * GH>(stage + kKeySteps + row0 * 4 * G + copy * 4 * GH, s0);
            load_shared<4 * GH>(stage + kKeySteps + row1 * 4 * G + copy * 4 * GH, s1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
#pragma unroll
            for (int j = 0; j < GH; ++j) {
                float c[NT][4] = {};
#pragma unroll
                for (int h = 0; h < COPIES; ++h) {
                    const int g = h * GH + j;
                    const uint32_t y[2] = {key_word(w0, g), key_word(w1, g)};
                    uint32_t ka[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t word = i ? y[e & 1] >> 8 : y[e & 1];
                            ka[i][e] = e < 2 ? masked_or<0x000f000fu>(word, f16_bits) : masked_or<0x00f000f0u>(word, f16_bits);
                            if constexpr (kExact) ka[i][e] = e < 2 ? centred_low(ka[i][e]) : centred_high(ka[i][e]);
                        }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int term = kTerms - 1; term >= 0; --term) {      // the largest terms last
                            mma_f16(c[n], ka[0], qb[term][n][g][0][0], qb[term][n][g][0][1]);
                            mma_f16(c[n], ka[1], qb[term][n][g][1][0], qb[term][n][g][1][1]);
                        }
                }
                const float step0 = __uint_as_float(s0[j] << 16), step1 = __uint_as_float(s1[j] << 16);
                float least0 = __uint_as_float(s0[j] & 0xffff0000u), least1 = __uint_as_float(s1[j] & 0xffff0000u);
                if constexpr (kExact) {
                    least0 = fmaf(8.0f, step0, least0);
                    least1 = fmaf(8.0f, step1, least1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (!kExact) c[n][e] -= q_offset[n][j][e & 1];
                        x[n][e] = fmaf(e < 2 ? step0 : step1, c[n][e], fmaf(e < 2 ? least0 : least1, q_sum[n][j][e & 1], x[n][e]));
                    }
            }
        }
        bool rises = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[n][e] = over_copies(x[n][e]) * to_log2[n][e & 1];
                if constexpr (EDGE) {
                    const int row = e < 2 ? row0 : row1, p = pos[n][e & 1];
                    const bool sees = ((seen >> row) & 1) && key0 + row <= p && (window == 0 || key0 + row > p - window);
                    x[n][e] = sees ? x[n][e] : -INFINITY;
                }
            }
            // The maximum moves only when a score passes it by more than 2^8: weights stay below 2^8, float32 and bfloat16 have room for them.
            rises |= fmaxf(x[n][0], x[n][2]) > top[n][0] + 8.0f || fmaxf(x[n][1], x[n][3]) > top[n][1] + 8.0f;
        }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(x[n][c], x[n][c + 2]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m, top[n][c]);
                    const float shrink = exp2_fast(top[n][c] - m);
                    top[n][c] = m;
                    total[n][c] *= shrink;
#pragma unroll
                    for (int g = 0; g < GH; ++g) least_sum[n][g][c] *= shrink;
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            o[n][g][u][c] *= shrink;
                            o[n][g][u][c + 2] *= shrink;
                        }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = exp2_fast(x[n][e] - top[n][e & 1]);
            total[n][0] += x[n][0] + x[n][2];
            total[n][1] += x[n][1] + x[n][3];
        }
        uint32_t s0[GH], s1[GH], va[G], vb[G], vc[G], vd[G];
        load_shared<4 * GH>(stage + kValueSteps + row0 * 4 * G + copy * 4 * GH, s0);
        load_shared<4 * GH>(stage + kValueSteps + row1 * 4 * G + copy * 4 * GH, s1);
        load_values(stage + kValues, placed(2 * t), r, va);
        load_values(stage + kValues, placed(2 * t + 1), r, vb);
        load_values(stage + kValues, placed(2 * t) + 8, r, vc);
        load_values(stage + kValues, placed(2 * t + 1) + 8, r, vd);
#pragma unroll
        for (int j = 0; j < GH; ++j) {
            const float step0 = __uint_as_float(s0[j] << 16), step1 = __uint_as_float(s1[j] << 16);
            const float middle0 = fmaf(8.0f, step0, __uint_as_float(s0[j] & 0xffff0000u)), middle1 = fmaf(8.0f, step1, __uint_as_float(s1[j] & 0xffff0000u));
            uint32_t b0[NT][kTerms], b1[NT][kTerms];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
                // EDGE: a weight of zero is nothing, whatever the value it belongs to
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = x[n][e] * (e < 2 ? step0 : step1);
                    if (EDGE && x[n][e] == 0.0f) w[e] = 0.0f;
                    else least_sum[n][j][e & 1] = fmaf(x[n][e], e < 2 ? middle0 : middle1, least_sum[n][j][e & 1]);
                }
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    b0[n][term] = transposed_8x8(pack_bf16(w[0], w[1]));
                    b1[n][term] = transposed_8x8(pack_bf16(w[2], w[3]));
                    if constexpr (kExact)
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] -= __bfloat162float(__float2bfloat16_rn(w[e]));
                }
            }
#pragma unroll
            for (int h = 0; h < COPIES; ++h) {
                const int g = h * GH + j;
                const uint32_t z0 = value_word(va, vb, g), z1 = value_word(vc, vd, g);
                uint32_t a0[4], a1[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t z = e < 2 ? z0 : z1;
                    a0[e] = centred(masked_or<0x000f000fu>(e % 2 ? z >> 4 : z, bf16_bits));
                    a1[e] = centred(masked_or<0x000f000fu>(e % 2 ? z >> 12 : z >> 8, bf16_bits));
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) {
                        mma_bf16(o[n][g][0], a0, b0[n][term], b1[n][term]);
                        mma_bf16(o[n][g][1], a1, b0[n][term], b1[n][term]);
                    }
            }
        }
    }
};

// Which rows of the pools a warp's turns are, and their copies into its ring.  Turn i of a warp is the keys key0 + i * kWarps4 * kTile4 .. + 15.
// Pages of whole turns: every turn is one run of rows.
template <typename B>
struct Turns16 {
    uint32_t units = kNoRow, units_next = kNoRow;         // of turns (32 n + lane) and the 32 behind them: row / 16
    uint32_t there = 0;                                   // bit i & 31: turn i has a page

    __device__ __forceinline__ uint32_t unit_of(const Attend4& a, const int* table, int kvh, int key) const {
        int logical, place;
        if (a.page_shift >= 0) {
            logical = key >> a.page_shift;
            place = key & (a.page_size - 1);
        } else {
            logical = key / a.page_size;
            place = key - logical * a.page_size;
        }
        const int page = table[logical];
        page_ok(page, a.bounds);
        return page_or_none(page, a.n_pages) < 0 ? kNoRow : (((uint32_t)page * a.Hkv + kvh) * a.page_size + place) / kTile4;
    }
    __device__ __forceinline__ uint32_t load(const Attend4& a, const int* table, int kvh, int key0, int turn, int own) const {
        return turn < own ? unit_of(a, table, kvh, key0 + turn * (kWarps4 * kTile4)) : kNoRow;
    }
    __device__ __forceinline__ void begin(const Attend4& a, const int* table, int kvh, int key0, int own, const Span4&, int lane) {
        units_next = load(a, table, kvh, key0, lane, own);
    }
    // Turn i, in order, into a stage.
    __device__ __forceinline__ void fill(const Attend4& a, const int* table, int kvh, int key0, int own, const Span4&, int i, uint32_t stage, int lane) {
        if ((i & 31) == 0) {
            units = units_next;
            units_next = load(a, table, kvh, key0, i + 32 + lane, own);
        }
        const uint32_t unit = __shfl_sync(0xffffffffu, units, i & 31);
        if (unit == kNoRow) {
            there &= ~(1u << (i & 31));
            return;
        }
        there |= 1u << (i & 31);
        const uint8_t* k = a.k.codes + (size_t)unit * (kTile4 * B::kRow) + lane * 16;
        const uint8_t* v = a.v.codes + (size_t)unit * (kTile4 * B::kRow) + lane * 16;
#pragma unroll
        for (int it = 0; it < (B::G_ + 1) / 2; ++it) {
            const int j = it * 32 + lane, key = j / B::G_, c = j - key * B::G_;
            if (B::G_ % 2 == 0 || j < kTile4 * B::G_) {
                const uint32_t to = stage + key * B::kRow + ((c ^ B::turned(key)) * 16);
                cp_async16(to, k + it * 512, true);
                cp_async16(to + B::kValues, v + it * 512, true);
            }
        }
#pragma unroll
        for (int it = 0; it < (8 * B::G_ + 31) / 32; ++it) {
            const int j = it * 32 + lane;
            const bool is_v = j >= 4 * B::G_;
            const int c = is_v ? j - 4 * B::G_ : j;
            if (8 * B::G_ % 32 == 0 || j < 8 * B::G_) {
                const uint8_t* steps = reinterpret_cast<const uint8_t*>(is_v ? a.v.steps : a.k.steps) + (size_t)unit * (kTile4 * 4 * B::G_) + c * 16;
                cp_async16(stage + (is_v ? B::kValueSteps : B::kKeySteps) + c * 16, steps, true);
            }
        }
    }
    __device__ __forceinline__ uint32_t seen(int i, uint32_t) const { return (there >> (i & 31)) & 1 ? 0xffffu : 0u; }
};

// Pages of any size: key by key.  `row`: of key (lane & 15) of the next turn.
template <typename B>
struct TurnsAny {
    uint32_t row = kNoRow;

    __device__ __forceinline__ uint32_t row_of(const Attend4& a, const int* table, int kvh, int key, const Span4& span) const {
        if (key < span.first || key > span.last) return kNoRow;
        const int logical = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size, page = table[logical];
        page_ok(page, a.bounds);
        return page_or_none(page, a.n_pages) < 0 ? kNoRow : ((uint32_t)page * a.Hkv + kvh) * a.page_size + (key - logical * a.page_size);
    }
    __device__ __forceinline__ void begin(const Attend4& a, const int* table, int kvh, int key0, int own, const Span4& span, int lane) {
        row = own > 0 ? row_of(a, table, kvh, key0 + (lane & 15), span) : kNoRow;
    }
    __device__ __forceinline__ void fill(const Attend4& a, const int* table, int kvh, int key0, int own, const Span4& span, int i, uint32_t stage, int lane) {
        const uint32_t bits = __ballot_sync(0xffffffffu, row != kNoRow) & 0xffffu;
        if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + B::kSeen), "r"(bits) : "memory");
#pragma unroll
        for (int it = 0; it < (B::G_ + 1) / 2; ++it) {
            const int j = it * 32 + lane, key = j / B::G_, c = j - key * B::G_;
            const uint32_t from = __shfl_sync(0xffffffffu, row, key & 15);
            if (B::G_ % 2 == 0 || j < kTile4 * B::G_) {
                const bool ok = from != kNoRow;
                const size_t at = ok ? from : 0;
                const uint32_t to = stage + key * B::kRow + ((c ^ B::turned(key)) * 16);
                cp_async16(to, a.k.codes + at * B::kRow + c * 16, ok);
                cp_async16(to + B::kValues, a.v.codes + at * B::kRow + c * 16, ok);
                cp_async4(stage + B::kKeySteps + j * 4, reinterpret_cast<const uint32_t*>(a.k.steps) + at * B::G_ + c, ok);
                cp_async4(stage + B::kValueSteps + j * 4, reinterpret_cast<const uint32_t*>(a.v.steps) + at * B::G_ + c, ok);
            }
        }
        row = i + 1 < own ? row_of(a, table, kvh, key0 + (i + 1) * (kWarps4 * kTile4) + (lane & 15), span) : kNoRow;
    }
    __device__ __forceinline__ uint32_t seen(int, uint32_t stage) const {
        uint32_t bits;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bits) : "r"(stage + B::kSeen));
        return bits;
    }
};

// Where row `local` (tokens times the kv head's query heads) of a sequence stands in q and out, as token * Hq + head; -1 behind the last.
__device__ __forceinline__ long row_at(const Attend4& a, int first_token, int n_tokens, int kvh, int local) {
    const int group = a.Hq / a.Hkv, token = local / group;
    return token < n_tokens && first_token + token < a.n_rows ? (long)(first_token + token) * a.Hq + kvh * group + (local - token * group) : -1;
}

template <typename T, int G, int NT, int COPIES, typename Turns, int BLOCKS>
__global__ void __launch_bounds__(kWarps4 * 32, BLOCKS) attend_4bit_kernel(const Attend4 a) {
    using B = Attend4Block<T, G, NT, COPIES>;
    constexpr int D = B::D;
    pdl_wait();
    extern __shared__ __align__(128) uint8_t shared[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
    const int part = blockIdx.x, kvh = blockIdx.y / a.row_blocks, row_block = blockIdx.y - kvh * a.row_blocks, seq = blockIdx.z;
    const int group = a.Hq / a.Hkv, row0 = row_block * B::kRows;
    const int first_token = a.cu_q ? a.cu_q[seq] : seq, n_tokens = a.cu_q ? a.cu_q[seq + 1] - first_token : 1, kv_len = a.kv_len[seq];
    if (row0 >= n_tokens * group) return;
    const int token0 = row0 / group, token1 = min(n_tokens - 1, (row0 + B::kRows - 1) / group);
    const Span4 span(a, kv_len, n_tokens, token0, token1);
    const int n_parts = span.parts(a);
    if (part >= n_parts && !(n_parts == 0 && part == 0)) return;
    const int begin = span.start() + part * a.part_keys, end = min(span.last + 1, begin + a.part_keys);
    const int tiles = end > begin ? (end - begin + kTile4 - 1) / kTile4 : 0, own = tiles > warp ? (tiles - warp + kWarps4 - 1) / kWarps4 : 0;

    const uint32_t ring = smem_u32(shared) + warp * B::kPerWarp;
    const int* table = a.table + (size_t)seq * a.width;
    const int key_first = begin + warp * kTile4;
    Turns turns;
    turns.begin(a, table, kvh, key_first, own, span, lane);
#pragma unroll
    for (int i = 0; i < kStages4 - 1; ++i) {
        if (i < own) turns.fill(a, table, kvh, key_first, own, span, i, ring + i * B::kStage, lane);
        cp_async_commit();
    }

    B b;
    const T* src[NT];
    int lowest = 0x7fffffff, highest = -0x7fffffff;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const long at = row_at(a, first_token, n_tokens, kvh, row0 + 8 * n + r % B::kColumns);
        src[n] = at < 0 ? nullptr : reinterpret_cast<const T*>(a.q) + at * D;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            b.pos[n][c] = min(span.last, kv_len - n_tokens + min(n_tokens - 1, (row0 + 8 * n + (2 * t + c) % B::kColumns) / group));
            b.top[n][c] = kLowest4;
            b.total[n][c] = 0.0f;
#pragma unroll
            for (int g = 0; g < B::GH; ++g) b.least_sum[n][g][c] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int u = 0; u < 2; ++u) b.o[n][g][u][c] = b.o[n][g][u][c + 2] = 0.0f;
        }
    }
    lowest = min(span.last, kv_len - n_tokens + token0);
    highest = kv_len - n_tokens + token1;
    b.load_q(src, a.scale_log2, lane);

    int stage = 0;
    for (int i = 0; i < own; ++i) {
        cp_async_wait<kStages4 - 2>();
        __syncwarp();
        const int next = i + kStages4 - 1, to = stage == 0 ? kStages4 - 1 : stage - 1;
        if (next < own) turns.fill(a, table, kvh, key_first, own, span, next, ring + to * B::kStage, lane);
        cp_async_commit();
        const uint32_t at = ring + stage * B::kStage, seen = turns.seen(i, at);
        const int key0 = key_first + i * (kWarps4 * kTile4);
        if (seen != 0xffffu || key0 + kTile4 - 1 > lowest || (a.window > 0 && key0 <= highest - a.window)) {
            if (seen != 0) b.template turn<true>(at, key0, seen, a.window, lane);
        } else {
            b.template turn<false>(at, key0, seen, a.window, lane);
        }
        stage = stage + 1 == kStages4 ? 0 : stage + 1;
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncwarp();
    pdl_trigger();

    // The warp's sums to its own shared memory (the ring is done with): [column][D], then maxima and totals.
    float* mine = reinterpret_cast<float*>(shared + warp * B::kPerWarp);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int column = 8 * n + (2 * t + c) % B::kColumns, copy = t * COPIES / 4;
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
            for (int g = 0; g < G; ++g) {
                const float m = least[g % B::GH];
                if (copy == g / B::GH)
                    *reinterpret_cast<float4*>(mine + column * D + 32 * g + 4 * r) =
                        make_float4(b.o[n][g][0][c] + m, b.o[n][g][0][c + 2] + m, b.o[n][g][1][c] + m, b.o[n][g][1][c + 2] + m);
            }
            if (r == 0 && copy == 0) {
                mine[B::kRows * D + 2 * column] = b.top[n][c];
                mine[B::kRows * D + 2 * column + 1] = total;
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < B::kRows * (D / 4); i += kWarps4 * 32) {
        const int column = i / (D / 4), quad = i - column * (D / 4);
        const long at = row_at(a, first_token, n_tokens, kvh, row0 + column);
        if (at < 0) continue;
        float tops[kWarps4], top = kLowest4, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
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
        if (a.parts == 1) {
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = total == 0.0f ? 0.0f : v[e] * inverse;
            store_quad(reinterpret_cast<T*>(a.out) + at * D + 4 * quad, v);
        } else {
            store_quad(a.sums + (at * a.parts + part) * D + 4 * quad, v);
            if (quad == 0) {
                float* ml = a.sums + (size_t)a.n_rows * a.Hq * a.parts * D + (at * a.parts + part) * 2;
                ml[0] = top;
                ml[1] = total;
            }
        }
    }
}

// The parts of a row joined: a warp a row.
template <typename T>
__global__ void join_4bit_kernel(const Attend4 a, int D, int rows_of_block) {
    pdl_wait();
    const int lane = threadIdx.x & 31, seq = blockIdx.y;
    const int first_token = a.cu_q ? a.cu_q[seq] : seq, n_tokens = a.cu_q ? a.cu_q[seq + 1] - first_token : 1;
    const int index = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), group = a.Hq / a.Hkv;
    if (index >= n_tokens * a.Hq) return;
    const int token = index / a.Hq, head = index - token * a.Hq, kvh = head / group, local = token * group + head - kvh * group;
    const int token0 = local / rows_of_block * rows_of_block / group, token1 = min(n_tokens - 1, (local / rows_of_block * rows_of_block + rows_of_block - 1) / group);
    const int used = Span4(a, a.kv_len[seq], n_tokens, token0, token1).parts(a);
    const long at = row_at(a, first_token, n_tokens, kvh, local);
    if (at < 0) return;
    const float* ml = a.sums + (size_t)a.n_rows * a.Hq * a.parts * D + at * a.parts * 2;
    float top = kLowest4, total = 0.0f, v[2][4] = {};
    for (int p = lane; p < used; p += 32) top = fmaxf(top, ml[2 * p]);
    top = warp_max(top);
    for (int p = lane; p < used; p += 32) total += exp2_fast(ml[2 * p] - top) * ml[2 * p + 1];
    total = warp_sum(total);
#pragma unroll 4
    for (int p = 0; p < used; ++p) {
        const float f = exp2_fast(ml[2 * p] - top);
        const float* s = a.sums + (at * a.parts + p) * D;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (4 * (lane + 32 * j) < D) {
                float w[4];
                load_quad(s + 4 * (lane + 32 * j), w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = fmaf(f, w[e], v[j][e]);
            }
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (4 * (lane + 32 * j) < D) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = total == 0.0f ? 0.0f : v[j][e] * inverse;
            store_quad(reinterpret_cast<T*>(a.out) + at * D + 4 * (lane + 32 * j), v[j]);
        }
}

template <typename T, int G, int NT, int COPIES, template <typename> class Turns>
int launch_attend_4bit(const Attend4& a, int most_tokens, cudaStream_t stream) {
    using B = Attend4Block<T, G, NT, COPIES>;
    constexpr int kRegs = G * NT * (4 * B::kTerms + 8) + 6 * NT * B::GH + 66;       // about: q, sums and the rest of a thread
    constexpr int kBlocks = kRegs <= 150 ? 4 : kRegs <= 180 ? 3 : 2;
    auto kernel = attend_4bit_kernel<T, G, NT, COPIES, Turns<B>, kBlocks>;
    static SmemLimit limit;
    if (const int rc = limit.allow(kernel, B::kShared)) return rc;
    if (const int rc = launch_pdl(kernel, dim3(a.parts, a.Hkv * a.row_blocks, a.n_seqs), dim3(kWarps4 * 32), B::kShared, stream, a)) return rc;
    if (a.parts == 1) return 0;
    return launch_pdl(join_4bit_kernel<T>, dim3((most_tokens * a.Hq + 3) / 4, a.n_seqs), dim3(128), 0, stream, a, B::D, B::kRows);
}

template <typename T, int G, template <typename> class Turns>
int launch_attend_4bit_of(const Attend4& a, int rows, int most_tokens, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (rows == 16) return launch_attend_4bit<T, G, 2, 1, Turns>(a, most_tokens, stream);
    if constexpr (G % 4 == 0)
        if (rows == 2) return launch_attend_4bit<T, G, 1, 4, Turns>(a, most_tokens, stream);
    if constexpr (G % 2 == 0)
        if (rows == 4) return launch_attend_4bit<T, G, 1, 2, Turns>(a, most_tokens, stream);
    return rows == 8 ? launch_attend_4bit<T, G, 1, 1, Turns>(a, most_tokens, stream) : PB_ERR_BAD_SIZE;
}

template <typename T, int G>
int launch_attend_4bit_of(const Attend4& a, int rows, int most_tokens, cudaStream_t stream) {
    return a.page_size % kTile4 == 0 ? launch_attend_4bit_of<T, G, Turns16>(a, rows, most_tokens, stream) : launch_attend_4bit_of<T, G, TurnsAny>(a, rows, most_tokens, stream);
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
