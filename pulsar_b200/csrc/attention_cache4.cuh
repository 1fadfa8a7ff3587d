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
// A code becomes a bfloat16 by one logical instruction for two of them: 128 + c is the bits 0x4300 | c.  A block takes one sequence, kv head,
// up to 8 NT rows (query heads of the kv head, tokens) and a part of the keys; its warps take runs of 16 keys in turn, each through a
// ring of its own in shared memory, so that nobody waits for anybody until the end.  mma.sync m16n8k16 has the keys in its 16 rows for
// the scores and the channels for the weighted sum, and the rows of the block in its 8 columns: with 4 or 8 query heads a kv head half of the
// products are wanted, where rows in its 16 would waste three quarters.  The weights change places between the two products by movmatrix.
// (tcgen05 would want codes as bfloat16 in shared memory, which is more traffic there than all the rest; what bounds this kernel are instructions
// on codes and bytes, not products.)
#pragma once

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
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
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
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// Codes e and e + 4 bits of both halves of a word, as 128 + c.
template <int NIBBLE> __device__ __forceinline__ uint32_t raw_codes(uint32_t word) { return ((word >> (4 * NIBBLE)) & 0x000f000fu) | 0x43004300u; }
// (128 + c) - 136 = c - 8, exactly.
__device__ __forceinline__ uint32_t centred(uint32_t raw) {
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&raw), __floats2bfloat162_rn(136.0f, 136.0f));
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

template <typename T, int G, int NT>
struct Attend4Block {
    static constexpr int D = kGroup4 * G;
    static constexpr bool kExact = sizeof(T) == 4;          // float32: operands of the products in three bfloat16 terms, codes about zero
    static constexpr int kTerms = kExact ? 3 : 1;
    static constexpr int kRow = 16 * G;                     // bytes of a row of codes
    static constexpr int kKeySteps = kTile4 * kRow, kValues = kKeySteps + kTile4 * 4 * G, kValueSteps = kValues + kTile4 * kRow;
    static constexpr int kSeen = kValueSteps + kTile4 * 4 * G, kStage = kSeen + 16;
    static constexpr int kRing = kStages4 * kStage;
    static constexpr int kMerge = (8 * NT * (D + 2) * 4 + 15) / 16 * 16;
    static constexpr int kPerWarp = kRing > kMerge ? kRing : kMerge;
    static constexpr int kShared = kWarps4 * kPerWarp;

    // Row k of 16 keys as the products number them stands in row placed(k) of a stage, and 16-byte chunk c of it at c ^ turned(row): the lanes of
    // either product then read different banks (heads of 128 and 256; the others have some conflicts).
    static __device__ __forceinline__ int placed(int k) { return k ^ ((k >> 1) & 1); }
    static __device__ __forceinline__ int turned(int row) { return G == 4 ? (row >> 1) & 2 : G == 8 ? row & 6 : 0; }

    static __device__ __forceinline__ uint32_t row_of(const Attend4& a, const int* table, int kvh, int key, const Span4& span) {
        if (key < span.first || key > span.last) return kNoRow;
        int logical, place;
        if (a.page_shift >= 0) {
            logical = key >> a.page_shift;
            place = key & (a.page_size - 1);
        } else {
            logical = key / a.page_size;
            place = key - logical * a.page_size;
        }
        if (logical >= a.width) return kNoRow;
        const int page = table[logical];
        page_ok(page, a.bounds);
        if (page_or_none(page, a.n_pages) < 0) return kNoRow;
        return ((uint32_t)page * a.Hkv + kvh) * a.page_size + place;
    }

    // Copies of 16 keys and values into a stage; `row` of a lane is that of key (lane & 15).  A key that is none gets zeros for its steps.
    static __device__ __forceinline__ void fill(const Attend4& a, uint32_t stage, uint32_t row, int lane) {
        const uint32_t seen = __ballot_sync(0xffffffffu, row != kNoRow) & 0xffffu;
        if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + kSeen), "r"(seen) : "memory");
#pragma unroll
        for (int it = 0; it < (G + 1) / 2; ++it) {
            const int i = it * 32 + lane, key = i / G, c = i - key * G;
            const uint32_t from = __shfl_sync(0xffffffffu, row, key & 15);
            if (G % 2 == 0 || i < kTile4 * G) {
                const bool ok = from != kNoRow;
                const size_t at = ok ? from : 0;
                const uint32_t code = key * kRow + ((c ^ turned(key)) * 16);
                cp_async16(stage + code, a.k.codes + at * kRow + c * 16, ok);
                cp_async16(stage + kValues + code, a.v.codes + at * kRow + c * 16, ok);
                cp_async4(stage + kKeySteps + i * 4, reinterpret_cast<const uint32_t*>(a.k.steps) + at * G + c, ok);
                cp_async4(stage + kValueSteps + i * 4, reinterpret_cast<const uint32_t*>(a.v.steps) + at * G + c, ok);
            }
        }
    }

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

    // State of a warp.  Lane (r, t) = (lane / 4, lane % 4) holds columns 2 t and 2 t + 1 of 8 rows of the block for each of NT.
    uint32_t qb[kTerms][NT][G][2][2];       // q as the second operand: column r, channels 32 g + 8 t + ..
    float q_sum[NT][G][2];                  // sum of a column's q over the group
    float o[NT][G][2][4];                   // [u]: channels 32 g + 4 r + 2 u, + 1 (elements 0 1, 2 3) of columns 2 t, 2 t + 1
    float least_sum[NT][G][2];              // this lane's part of sum_j p_j (m_j + 8 s_j)
    float top[NT][2], total[NT][2];
    int pos[NT][2];                         // a column's position

    __device__ __forceinline__ void load_q(const T* const (&src)[NT], int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float v[8];
                const int t = lane & 3;
                if (src[n] != nullptr) {
                    load_quad(src[n] + 32 * g + 8 * t, *reinterpret_cast<float(*)[4]>(v));
                    load_quad(src[n] + 32 * g + 8 * t + 4, *reinterpret_cast<float(*)[4]>(v + 4));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                }
                float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                q_sum[n][g][0] = __shfl_sync(0xffffffffu, s, 8 * t);
                q_sum[n][g][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) qb[term][n][g][h][e] = pack_bf16(v[2 * h + e], v[4 + 2 * h + e]);
                    if constexpr (kExact)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] -= __bfloat162float(__float2bfloat16_rn(v[e]));
                }
            }
    }

    // Sixteen keys.  EDGE: some column does not see some of them.
    template <bool EDGE>
    __device__ __forceinline__ void turn(uint32_t stage, int key0, uint32_t seen, float scale_log2, int window, int lane) {
        const int r = lane >> 2, t = lane & 3, row0 = placed(r), row1 = row0 + 8;
        float x[NT][4];
        {
            uint32_t w0[G], w1[G], s0[G], s1[G];
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
            load_shared<4 * G>(stage + kKeySteps + row0 * 4 * G, s0);
            load_shared<4 * G>(stage + kKeySteps + row1 * 4 * G, s1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t y0 = key_word(w0, g), y1 = key_word(w1, g);
                uint32_t ka[2][4] = {{raw_codes<0>(y0), raw_codes<0>(y1), raw_codes<1>(y0), raw_codes<1>(y1)},
                                     {raw_codes<2>(y0), raw_codes<2>(y1), raw_codes<3>(y0), raw_codes<3>(y1)}};
                float step0 = __uint_as_float(s0[g] << 16), least0 = __uint_as_float(s0[g] & 0xffff0000u);
                float step1 = __uint_as_float(s1[g] << 16), least1 = __uint_as_float(s1[g] & 0xffff0000u);
                if constexpr (kExact) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) ka[h][e] = centred(ka[h][e]);
                    least0 = fmaf(8.0f, step0, least0);
                    least1 = fmaf(8.0f, step1, least1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float c[4];
                    // sum q (128 + c) begins at -128 sum q
                    const float c0 = kExact ? 0.0f : -128.0f * q_sum[n][g][0], c1 = kExact ? 0.0f : -128.0f * q_sum[n][g][1];
                    mma_from(c, ka[0], qb[kTerms - 1][n][g][0][0], qb[kTerms - 1][n][g][0][1], c0, c1);
                    mma_bf16(c, ka[1], qb[kTerms - 1][n][g][1][0], qb[kTerms - 1][n][g][1][1]);
#pragma unroll
                    for (int term = kTerms - 2; term >= 0; --term) {          // the largest terms last
                        mma_bf16(c, ka[0], qb[term][n][g][0][0], qb[term][n][g][0][1]);
                        mma_bf16(c, ka[1], qb[term][n][g][1][0], qb[term][n][g][1][1]);
                    }
                    x[n][0] = fmaf(step0, c[0], fmaf(least0, q_sum[n][g][0], x[n][0]));
                    x[n][1] = fmaf(step0, c[1], fmaf(least0, q_sum[n][g][1], x[n][1]));
                    x[n][2] = fmaf(step1, c[2], fmaf(least1, q_sum[n][g][0], x[n][2]));
                    x[n][3] = fmaf(step1, c[3], fmaf(least1, q_sum[n][g][1], x[n][3]));
                }
            }
        }
        bool rises = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[n][e] *= scale_log2;
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
                    for (int g = 0; g < G; ++g) {
                        least_sum[n][g][c] *= shrink;
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            o[n][g][u][c] *= shrink;
                            o[n][g][u][c + 2] *= shrink;
                        }
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
        uint32_t s0[G], s1[G], va[G], vb[G], vc[G], vd[G];
        load_shared<4 * G>(stage + kValueSteps + row0 * 4 * G, s0);
        load_shared<4 * G>(stage + kValueSteps + row1 * 4 * G, s1);
        load_values(stage + kValues, placed(2 * t), r, va);
        load_values(stage + kValues, placed(2 * t + 1), r, vb);
        load_values(stage + kValues, placed(2 * t) + 8, r, vc);
        load_values(stage + kValues, placed(2 * t + 1) + 8, r, vd);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t z0 = value_word(va, vb, g), z1 = value_word(vc, vd, g);
            const uint32_t a0[4] = {centred(raw_codes<0>(z0)), centred(raw_codes<1>(z0)), centred(raw_codes<0>(z1)), centred(raw_codes<1>(z1))};
            const uint32_t a1[4] = {centred(raw_codes<2>(z0)), centred(raw_codes<3>(z0)), centred(raw_codes<2>(z1)), centred(raw_codes<3>(z1))};
            const float step0 = __uint_as_float(s0[g] << 16), step1 = __uint_as_float(s1[g] << 16);
            const float middle0 = fmaf(8.0f, step0, __uint_as_float(s0[g] & 0xffff0000u)), middle1 = fmaf(8.0f, step1, __uint_as_float(s1[g] & 0xffff0000u));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
                // EDGE: a weight of zero is nothing, whatever the value it belongs to
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = x[n][e] * (e < 2 ? step0 : step1);
                    if (EDGE && x[n][e] == 0.0f) w[e] = 0.0f;
                    else least_sum[n][g][e & 1] = fmaf(x[n][e], e < 2 ? middle0 : middle1, least_sum[n][g][e & 1]);
                }
                uint32_t b0[kTerms], b1[kTerms];
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    b0[term] = transposed_8x8(pack_bf16(w[0], w[1]));
                    b1[term] = transposed_8x8(pack_bf16(w[2], w[3]));
                    if constexpr (kExact)
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] -= __bfloat162float(__float2bfloat16_rn(w[e]));
                }
#pragma unroll
                for (int term = kTerms - 1; term >= 0; --term) {
                    mma_bf16(o[n][g][0], a0, b0[term], b1[term]);
                    mma_bf16(o[n][g][1], a1, b0[term], b1[term]);
                }
            }
        }
    }
};

// Where row `local` (tokens times the kv head's query heads) of a sequence stands in q and out, as token * Hq + head; -1 behind the last.
__device__ __forceinline__ long row_at(const Attend4& a, int first_token, int n_tokens, int kvh, int local) {
    const int group = a.Hq / a.Hkv, token = local / group;
    return token < n_tokens && first_token + token < a.n_rows ? (long)(first_token + token) * a.Hq + kvh * group + (local - token * group) : -1;
}

template <typename T, int G, int NT, int BLOCKS>
__global__ void __launch_bounds__(kWarps4 * 32, BLOCKS) attend_4bit_kernel(const Attend4 a) {
    using B = Attend4Block<T, G, NT>;
    constexpr int D = B::D;
    pdl_wait();
    extern __shared__ __align__(128) uint8_t shared[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
    const int part = blockIdx.x, kvh = blockIdx.y / a.row_blocks, row_block = blockIdx.y - kvh * a.row_blocks, seq = blockIdx.z;
    const int group = a.Hq / a.Hkv, row0 = row_block * 8 * NT;
    const int first_token = a.cu_q ? a.cu_q[seq] : seq, n_tokens = a.cu_q ? a.cu_q[seq + 1] - first_token : 1, kv_len = a.kv_len[seq];
    if (row0 >= n_tokens * group) return;
    const int token0 = row0 / group, token1 = min(n_tokens - 1, (row0 + 8 * NT - 1) / group);
    const Span4 span(a, kv_len, n_tokens, token0, token1);
    const int n_parts = span.parts(a);
    if (part >= n_parts && !(n_parts == 0 && part == 0)) return;
    const int begin = span.start() + part * a.part_keys, end = min(span.last + 1, begin + a.part_keys);
    const int tiles = end > begin ? (end - begin + kTile4 - 1) / kTile4 : 0, own = tiles > warp ? (tiles - warp + kWarps4 - 1) / kWarps4 : 0;

    const uint32_t ring = smem_u32(shared) + warp * B::kPerWarp;
    const int* table = a.table + (size_t)seq * a.width;
    const int key_of_lane = begin + warp * kTile4 + (lane & 15);
    uint32_t row = B::row_of(a, table, kvh, own > 0 ? key_of_lane : -1, span);
#pragma unroll
    for (int i = 0; i < kStages4 - 1; ++i) {
        if (i < own) B::fill(a, ring + i * B::kStage, row, lane);
        cp_async_commit();
        row = i + 1 < own ? B::row_of(a, table, kvh, key_of_lane + (i + 1) * kWarps4 * kTile4, span) : kNoRow;
    }

    B b;
    const T* src[NT];
    int lowest = 0x7fffffff, highest = -0x7fffffff;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const long at = row_at(a, first_token, n_tokens, kvh, row0 + 8 * n + r);
        src[n] = at < 0 ? nullptr : reinterpret_cast<const T*>(a.q) + at * D;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            b.pos[n][c] = kv_len - n_tokens + min(n_tokens - 1, (row0 + 8 * n + 2 * t + c) / group);
            b.top[n][c] = kLowest4;
            b.total[n][c] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                b.least_sum[n][g][c] = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u) b.o[n][g][u][c] = b.o[n][g][u][c + 2] = 0.0f;
            }
        }
    }
    lowest = kv_len - n_tokens + token0;
    highest = kv_len - n_tokens + token1;
    b.load_q(src, lane);

    int stage = 0;
    for (int i = 0; i < own; ++i) {
        cp_async_wait<kStages4 - 2>();
        __syncwarp();
        const int next = i + kStages4 - 1, to = stage == 0 ? kStages4 - 1 : stage - 1;
        if (next < own) B::fill(a, ring + to * B::kStage, row, lane);
        cp_async_commit();
        row = next + 1 < own ? B::row_of(a, table, kvh, key_of_lane + (next + 1) * kWarps4 * kTile4, span) : kNoRow;
        const uint32_t at = ring + stage * B::kStage;
        const int key0 = begin + (warp + i * kWarps4) * kTile4;
        uint32_t seen;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(seen) : "r"(at + B::kSeen));
        if (seen != 0xffffu || key0 + kTile4 - 1 > lowest || (a.window > 0 && key0 <= highest - a.window))
            b.template turn<true>(at, key0, seen, a.scale_log2, a.window, lane);
        else
            b.template turn<false>(at, key0, seen, a.scale_log2, a.window, lane);
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
            const int column = 8 * n + 2 * t + c;
            float total = b.total[n][c];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float least = b.least_sum[n][g][c];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) least += __shfl_xor_sync(0xffffffffu, least, off);
                const float4 v = make_float4(b.o[n][g][0][c] + least, b.o[n][g][0][c + 2] + least, b.o[n][g][1][c] + least, b.o[n][g][1][c + 2] + least);
                *reinterpret_cast<float4*>(mine + column * D + 32 * g + 4 * r) = v;
            }
            if (r == 0) {
                mine[8 * NT * D + 2 * column] = b.top[n][c];
                mine[8 * NT * D + 2 * column + 1] = total;
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * NT * (D / 4); i += kWarps4 * 32) {
        const int column = i / (D / 4), quad = i - column * (D / 4);
        const long at = row_at(a, first_token, n_tokens, kvh, row0 + column);
        if (at < 0) continue;
        float tops[kWarps4], top = kLowest4, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWarps4; ++w) {
            tops[w] = reinterpret_cast<const float*>(shared + w * B::kPerWarp)[8 * NT * D + 2 * column];
            top = fmaxf(top, tops[w]);
        }
#pragma unroll
        for (int w = 0; w < kWarps4; ++w) {
            const float* theirs = reinterpret_cast<const float*>(shared + w * B::kPerWarp);
            const float f = exp2_fast(tops[w] - top);
            const float4 s = *reinterpret_cast<const float4*>(theirs + column * D + 4 * quad);
            total += f * theirs[8 * NT * D + 2 * column + 1];
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

template <typename T, int G, int NT>
int launch_attend_4bit(const Attend4& a, int most_tokens, cudaStream_t stream) {
    using B = Attend4Block<T, G, NT>;
    constexpr int kRegs = 4 * G * NT * (2 * B::kTerms + 2) + 2 * NT * G + 70;       // about: q, sums and the rest of a thread
    constexpr int kBlocks = kRegs <= 126 ? 4 : kRegs <= 160 ? 3 : 2;
    auto kernel = attend_4bit_kernel<T, G, NT, kBlocks>;
    static SmemLimit limit;
    if (const int rc = limit.allow(kernel, B::kShared)) return rc;
    if (const int rc = launch_pdl(kernel, dim3(a.parts, a.Hkv * a.row_blocks, a.n_seqs), dim3(kWarps4 * 32), B::kShared, stream, a)) return rc;
    if (a.parts == 1) return 0;
    return launch_pdl(join_4bit_kernel<T>, dim3((most_tokens * a.Hq + 3) / 4, a.n_seqs), dim3(128), 0, stream, a, B::D, 8 * NT);
}

template <typename T, int NT>
int launch_attend_4bit_of(const Attend4& a, int groups, int most_tokens, cudaStream_t stream) {
    switch (groups) {
        case 1: return launch_attend_4bit<T, 1, NT>(a, most_tokens, stream);
        case 2: return launch_attend_4bit<T, 2, NT>(a, most_tokens, stream);
        case 3: return launch_attend_4bit<T, 3, NT>(a, most_tokens, stream);
        case 4: return launch_attend_4bit<T, 4, NT>(a, most_tokens, stream);
        case 5: return launch_attend_4bit<T, 5, NT>(a, most_tokens, stream);
        case 6: return launch_attend_4bit<T, 6, NT>(a, most_tokens, stream);
        case 7: return launch_attend_4bit<T, 7, NT>(a, most_tokens, stream);
        case 8: return launch_attend_4bit<T, 8, NT>(a, most_tokens, stream);
    }
    return PB_ERR_BAD_SIZE;
}

int attend_4bit_f32(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream);      // rows of a block: 8 or 16
int attend_4bit_bf16(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream);

}  // namespace pb
