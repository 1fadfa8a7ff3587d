// Keys and values into a cache of 4 bits, and back (cache4.cuh has the format).
//
//   qk_norm_rope_write_4bit   per (token, head) of a projection row [q: Hq*D | k: Hkv*D | v: Hkv*D]: q and k are normed (x / sqrt(mean(x^2) + eps) * w,
//                             where weights are given) and their first `rotary` channels turned, (u, v) -> (u cos - v sin, v cos + u sin)
//                             with v half a turn's width behind u; q is rounded to T, k and v to T and then to 4 bits, at their slots.  (q in 32 bits, as
//                             much as its scores have; k in 64, because a rounding more may move a code.)
//   expand_pages_4bit         the values of the pages that sequences hold, as T, into pages of their own.
#include "cache4.cuh"

namespace {

using namespace pb;

__device__ __forceinline__ float root_inverse(float v) { return rsqrtf(v); }
__device__ __forceinline__ double root_inverse(double v) { return rsqrt(v); }
template <typename A> __device__ __forceinline__ A sum_of_warp(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A lane's quads of a head, channels 4 (lane + 32 j) .. + 3: normed and turned with arithmetic in A.  `shared`: D numbers of this warp.
template <typename A, typename T, int QUADS>
__device__ __forceinline__ void norm_and_turn(const T* __restrict__ src, const float* __restrict__ weight, double eps, const float* __restrict__ cos_t,
                                              const float* __restrict__ sin_t, int D, int rotary, int lane, A* shared, A (&x)[QUADS][4]) {
    A ss = 0;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const int at = 4 * (lane + 32 * j);
        float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (at < D) load_quad(src + at, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[j][e] = (A)f[e];
            ss += x[j][e] * x[j][e];
        }
    }
    if (weight != nullptr) {
        const A r = root_inverse(sum_of_warp(ss) / (A)D + (A)eps);
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const int at = 4 * (lane + 32 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at < D) x[j][e] = x[j][e] * r * (A)weight[at + e];
        }
    }
    if (rotary == 0) return;
    const int half = rotary >> 1;
#pragma unroll
    for (int j = 0; j < QUADS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * (lane + 32 * j) < D) shared[4 * (lane + 32 * j) + e] = x[j][e];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < QUADS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 4 * (lane + 32 * j) + e;
            if (i < half) x[j][e] = x[j][e] * (A)cos_t[i] - shared[i + half] * (A)sin_t[i];
            else if (i < rotary) x[j][e] = x[j][e] * (A)cos_t[i - half] + shared[i - half] * (A)sin_t[i - half];
        }
}

// A lane's four values of a group, eight lanes a group, to codes and steps at row `at` of a pool.  The steps and codes are found in 64 bits: a
// value next to the border of two codes falls where the formula has it.
__device__ __forceinline__ void quantise_quad(const float (&y)[4], int quad, int own, int groups, size_t at, const Pool4& pool) {
    float lo = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])), hi = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!(fabsf(y[e]) <= kMost4)) hi = __int_as_float(0x7f800000);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (4 * quad >= kGroup4 * own) return;              // a lane without channels
    const bool bad = hi > kMost4;
    const double m = (double)__bfloat162float(__float2bfloat16_rd(lo));
    // A quotient is a product with the reciprocal r and Newton's step for what is left, q + (d - q b) r, which leaves the square of r's error: below what 64
    // bits hold, so that a quotient that they hold exactly (a tie between two codes) comes out as that.  The reciprocal of a step is that of 32 bits after one
    // such step of its own; of steps whose reciprocal 32 bits do not hold, a division's.
    constexpr double kFifteenth = 1.0 / 15.0;
    const double range = (double)hi - m, rough = range * kFifteenth;
    const float step = __bfloat162float(__float2bfloat16_ru(__double2float_ru(fma(fma(-rough, 15.0, range), kFifteenth, rough))));
    const double s = (double)step;
    double inverse = (double)__frcp_rn(step);
    inverse = fma(fma(-s, inverse, 1.0), inverse, inverse);
    if (!(step > 1e-37f && step < 1e37f)) inverse = step > 0.0f ? 1.0 / s : 0.0;
    uint32_t word = 0;
    if (!bad) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double d = (double)y[e] - m;
            double c = d * inverse;
            c = fma(fma(-c, s, d), inverse, c);
            word |= (uint32_t)min(15, __double2int_rn(c)) << (4 * e);
        }
    }
    const int g = quad >> 3, r = quad & 7;
    reinterpret_cast<uint16_t*>(pool.codes)[at * (size_t)(groups * 8) + r * groups + g] = (uint16_t)word;
    if (r == 0) {
        const uint32_t two = (__float_as_uint(step) >> 16) | (__float_as_uint((float)m) & 0xffff0000u);
        reinterpret_cast<uint32_t*>(pool.steps)[at * (size_t)groups + g] = bad ? 0x7fc07fc0u : two;
    }
}

template <typename T, int QUADS>
__global__ void qk_norm_rope_write_4bit_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, Pool4 k_pool, Pool4 v_pool, const int* __restrict__ slots,
                                               const float* __restrict__ cos_t, const float* __restrict__ sin_t, const float* __restrict__ q_weight,
                                               const float* __restrict__ k_weight, double eps, int Hq, int Hkv, int D, int rotary, int page_size, int n_pages,
                                               const PoolBounds bounds) {
    pdl_wait();
    extern __shared__ __align__(16) double shared[];         // [warps][D]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
    const int head = blockIdx.y * (blockDim.x >> 5) + warp;
    if (head >= Hq + 2 * Hkv) return;
    const T* src = qkv + ((size_t)t * (Hq + 2 * Hkv) + head) * D;
    const float* c = cos_t + (size_t)t * (rotary >> 1);
    const float* s = sin_t + (size_t)t * (rotary >> 1);
    if (head < Hq) {
        float x[QUADS][4];
        norm_and_turn<float>(src, q_weight, eps, c, s, D, rotary, lane, reinterpret_cast<float*>(shared + (size_t)warp * D), x);
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
            if (4 * (lane + 32 * j) < D) store_quad(q_out + ((size_t)t * Hq + head) * D + 4 * (lane + 32 * j), x[j]);
        return;
    }
    const int slot = slots[t];
    if (slot < 0 || !slot_ok(slot, page_size, bounds) || page_or_none(slot / page_size, n_pages) < 0) return;
    const bool is_k = head < Hq + Hkv;
    const int h = is_k ? head - Hq : head - Hq - Hkv;
    const size_t at = ((size_t)(slot / page_size) * Hkv + h) * page_size + slot % page_size;
    const Pool4 pool = {is_k ? k_pool.codes : v_pool.codes, is_k ? k_pool.steps : v_pool.steps};
    float y[QUADS][4] = {};
    if (is_k) {
        double x[QUADS][4];
        norm_and_turn<double>(src, k_weight, eps, c, s, D, rotary, lane, shared + (size_t)warp * D, x);
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[j][e] = to_float(from_float<T>((float)x[j][e]));
    } else {
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
            if (4 * (lane + 32 * j) < D) load_quad(src + 4 * (lane + 32 * j), y[j]);
    }
#pragma unroll
    for (int j = 0; j < QUADS; ++j) quantise_quad(y[j], lane + 32 * j, D / kGroup4, D / kGroup4, at, pool);
}

// qk_norm_rope_write_4bit where a head is 8, 16 or 32 lanes of four channels of its first half and the same four of its second, and all of them turn, or
// none: both ends of a turn are in one lane, as many heads a warp as fit, a group in eight lanes.  What bounds it are instructions (issue slots 71 % full,
// conversions to and from 64 bits 40 % of their unit): 2,048 bfloat16 tokens of 32 / 8 heads of 128 take 18.5 us, where their bytes would take 7; one
// token 2.3.  The kernel above, which takes every other size, takes 41 and 3.3 for them.  (Tried: several tokens a block, 24 where it was 19; twelve blocks an SM
// instead of ten, 20.)
template <int L, typename A> __device__ __forceinline__ A sum_of_lanes(A v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ void store_octet(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_octet(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct Turn4 {
    float w[2][4], c[4], s[4];
    bool norm, turns;
    template <int L> __device__ __forceinline__ void load_weight(const float* __restrict__ weight, int l) {
        norm = weight != nullptr;
        if (norm) {
            load_quad(weight + 4 * l, w[0]);
            load_quad(weight + 4 * (L + l), w[1]);
        }
    }
};
template <typename A, int L>
__device__ __forceinline__ void norm_and_turn_pair(const float (&f)[2][4], const Turn4& t, double eps, A (&x)[2][4]) {
    A ss = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[i][e] = (A)f[i][e];
            if (t.norm) ss += x[i][e] * x[i][e];
        }
    if (t.norm) {
        const A r = root_inverse(sum_of_lanes<L>(ss) / (A)(8 * L) + (A)eps);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = x[i][e] * r * (A)t.w[i][e];
    }
    if (!t.turns) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const A u = x[0][e], v = x[1][e];
        x[0][e] = u * (A)t.c[e] - v * (A)t.s[e];
        x[1][e] = v * (A)t.c[e] + u * (A)t.s[e];
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(128, 10) write_lanes_4bit_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, Pool4 k_pool, Pool4 v_pool, const int* __restrict__ slots,
                                                               const float* __restrict__ cos_t, const float* __restrict__ sin_t, const float* __restrict__ q_weight,
                                                               const float* __restrict__ k_weight, double eps, int Hq, int Hkv, int turns, int page_size, int n_pages,
                                                               const PoolBounds bounds) {
    pdl_wait();
    constexpr int D = kGroup4 * G, L = D / 8;
    const int l = threadIdx.x & (L - 1);
    // a block is of queries, keys or values alone; lanes of heads that there are not only keep their neighbours company
    constexpr int kHeads = 128 / L;
    const int kv_blocks = (Hkv + kHeads - 1) / kHeads;                  // keys first: their blocks take longest
    const int section = (int)blockIdx.y < kv_blocks ? 1 : (int)blockIdx.y < 2 * kv_blocks ? 2 : 0;
    const int h = ((int)blockIdx.y - (section == 1 ? 0 : section == 2 ? kv_blocks : 2 * kv_blocks)) * kHeads + threadIdx.x / L;
    const bool there = h < (section == 0 ? Hq : Hkv);
    const int head = (there ? h : 0) + (section == 0 ? 0 : section == 1 ? Hq : Hq + Hkv);
    const Pool4 pool = {section == 1 ? k_pool.codes : v_pool.codes, section == 1 ? k_pool.steps : v_pool.steps};
    Turn4 turn;
    turn.turns = section < 2 && turns;
    turn.load_weight<L>(section == 0 ? q_weight : section == 1 ? k_weight : nullptr, l);
    const int t = blockIdx.x;
    float y[2][4];
    const T* src = qkv + ((size_t)t * (Hq + 2 * Hkv) + head) * D + 4 * l;
    load_quad(src, y[0]);
    load_quad(src + D / 2, y[1]);
    if (turn.turns) {
        load_quad(cos_t + (size_t)t * (D / 2) + 4 * l, turn.c);
        load_quad(sin_t + (size_t)t * (D / 2) + 4 * l, turn.s);
    }
    if (section == 0) {
        float x[2][4];
        norm_and_turn_pair<float, L>(y, turn, eps, x);
        T* dst = q_out + ((size_t)t * Hq + h) * D + 4 * l;
        if (there) {
            store_quad(dst, x[0]);
            store_quad(dst + D / 2, x[1]);
        }
        return;
    }
    const int slot = slots[t];
    if (slot < 0 || !slot_ok(slot, page_size, bounds) || page_or_none(slot / page_size, n_pages) < 0) return;
    const size_t at = ((size_t)(slot / page_size) * Hkv + h) * page_size + slot % page_size;
    if (section == 1) {
        double x[2][4];
        norm_and_turn_pair<double, L>(y, turn, eps, x);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][e] = to_float(from_float<T>((float)x[i][e]));
    }
    quantise_quad(y[0], l, there ? G : 0, G, at, pool);
    quantise_quad(y[1], L + l, there ? G : 0, G, at, pool);
}

// N neighbouring words, aligned to as many of them as make 16, 8 or 4 bytes.
template <int N> __device__ __forceinline__ void load_words(const uint32_t* __restrict__ p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = *reinterpret_cast<const uint4*>(p + 4 * i);
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) *reinterpret_cast<uint2*>(w + 2 * i) = *reinterpret_cast<const uint2*>(p + 2 * i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = p[i];
    }
}

// A lane's 8 G codes of a row, channels 8 t .. + 7 of every group, as values that lie at most `most` from zero.
template <bool BOUNDED, typename T, int G>
__device__ __forceinline__ void store_values(const uint32_t (&w)[G], const uint32_t (&two)[G], T* dst, float most) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float step = __uint_as_float(two[g] << 16), least = __uint_as_float(two[g] & 0xffff0000u);
        // 16-bit words g and G + g of the lane's 2 G
        const uint32_t sel = ((g & 1) ? 0x0032u : 0x0010u) | (((G + g) & 1) ? 0x7600u : 0x5400u), word = __byte_perm(w[g >> 1], w[(G + g) >> 1], sel);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            y[e] = fmaf(step, __uint_as_float(((word >> (4 * e)) & 15) | 0x4b000000u) - 8388608.0f, least);
            if (BOUNDED) y[e] = fminf(fmaxf(y[e], -most), most);
        }
        store_octet(dst + 32 * g, y);
    }
}
template <typename T, int G> __device__ __forceinline__ void store_zeros(T* dst) {
    const float zero[8] = {};
#pragma unroll
    for (int g = 0; g < G; ++g) store_octet(dst + 32 * g, zero);
}

// A lane takes the codes of channels 8 t .. + 7 of all groups of a row, side by side in the pool, and writes eight values of every group.  Bytes bound it: 5
// sequences of 15,000 to 30,000 bfloat16 keys, 8 heads of 128, take 95 us at 6.1 TB/s, three quarters of them written.
template <typename T, int G>
__global__ void __launch_bounds__(256) expand_pages_4bit_kernel(Pool4 k_pool, Pool4 v_pool, const int* __restrict__ table, const int* __restrict__ kv_len,
                                                                T* __restrict__ k_out, T* __restrict__ v_out, int* __restrict__ table_out, int width, int Hkv,
                                                                int page_size, int n_pages, const PoolBounds bounds) {
    pdl_wait();
    constexpr int D = kGroup4 * G;
    const int seq = blockIdx.y, logical = blockIdx.x, length = kv_len[seq];
    const size_t out_page = (size_t)seq * width + logical;
    const int rows = min(page_size, length - logical * page_size);              // of this page, that hold a key
    const int page = rows > 0 ? table[(size_t)seq * width + logical] : -1;
    if (rows > 0 && page >= 0) page_ok(page, bounds);
    const bool there = page_or_none(page, n_pages) >= 0;
    if (blockIdx.z == 0 && threadIdx.x == 0) table_out[out_page] = there ? (int)out_page : -1;
    if (!there) return;
    const int per_pool = Hkv * page_size, n = 2 * per_pool * 4;
    const bool partly = rows < page_size;
    for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < n; i += gridDim.z * blockDim.x) {
        const int t = i & 3, both = i >> 2;
        const bool is_v = both >= per_pool;
        const int row = is_v ? both - per_pool : both;                          // head * page_size + place
        const Pool4 pool = {is_v ? v_pool.codes : k_pool.codes, is_v ? v_pool.steps : k_pool.steps};
        T* dst = (is_v ? v_out : k_out) + (out_page * per_pool + row) * D + 8 * t;
        if (partly && row % page_size >= rows) {
            store_zeros<T, G>(dst);
            continue;
        }
        const size_t in_pool = (size_t)page * per_pool + row;
        uint32_t w[G], two[G];
        load_words<G>(reinterpret_cast<const uint32_t*>(pool.codes) + (in_pool * 4 + t) * G, w);
        load_words<G>(reinterpret_cast<const uint32_t*>(pool.steps) + in_pool * G, two);
        store_values<false, T, G>(w, two, dst, 0.0f);
    }
}

// The same for the dense attention kernels: a page that no tile of 128 keys touches which a query sees is left out, and what else is none becomes zeros.
// Those kernels want every value finite, seen or not, for a weight of zero times a NaN is one, in every row of the tile and of the tiles that find it
// in their buffers later; scores of keys that a row does not see they take away whatever those are.  So the key of a value that is no number becomes NaN
// and the value finite: who sees it gets NaN, and nobody else.  A lane takes a key and its value.
template <int G>
__global__ void __launch_bounds__(256) expand_for_attention_4bit_kernel(Pool4 k_pool, Pool4 v_pool, const int* __restrict__ table, const int* __restrict__ kv_len,
                                                                        __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                                                                        int* __restrict__ table_out, int width, int Hkv, int page_size, int n_pages,
                                                                        const int* __restrict__ cu_q, int window, const PoolBounds bounds) {
    pdl_wait();
    constexpr int D = kGroup4 * G;
    const int seq = blockIdx.y, logical = blockIdx.x, length = kv_len[seq];
    const size_t out_page = (size_t)seq * width + logical;
    const int low = window > 0 ? length - (cu_q[seq + 1] - cu_q[seq]) - window + 1 - 128 : 0;
    const bool there = logical * page_size < length && (logical + 1) * page_size > low;
    if (blockIdx.z == 0 && threadIdx.x == 0) table_out[out_page] = there ? (int)out_page : -1;
    if (!there) return;
    const int page = table[out_page];
    if (page >= 0) page_ok(page, bounds);
    const int rows = page_or_none(page, n_pages) >= 0 ? min(page_size, length - logical * page_size) : 0;      // of this page, that hold a key
    const int per_pool = Hkv * page_size, n = per_pool * 4;
    const bool partly = rows < page_size;
    for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < n; i += gridDim.z * blockDim.x) {
        const int t = i & 3, row = i >> 2;                                      // head * page_size + place
        const size_t to = (out_page * per_pool + row) * D + 8 * t;
        if (partly && row % page_size >= rows) {
            store_zeros<__nv_bfloat16, G>(k_out + to);
            store_zeros<__nv_bfloat16, G>(v_out + to);
            continue;
        }
        const size_t in_pool = (size_t)page * per_pool + row;
        uint32_t k[G], v[G], k_two[G], v_two[G];
        load_words<G>(reinterpret_cast<const uint32_t*>(k_pool.codes) + (in_pool * 4 + t) * G, k);
        load_words<G>(reinterpret_cast<const uint32_t*>(k_pool.steps) + in_pool * G, k_two);
        load_words<G>(reinterpret_cast<const uint32_t*>(v_pool.codes) + (in_pool * 4 + t) * G, v);
        load_words<G>(reinterpret_cast<const uint32_t*>(v_pool.steps) + in_pool * G, v_two);
        bool bounded = false;                   // a value passes the end of bfloat16's range, or is none
#pragma unroll
        for (int g = 0; g < G; ++g)
            bounded |= !(fmaf(15.0f, fabsf(__uint_as_float(v_two[g] << 16)), fabsf(__uint_as_float(v_two[g] & 0xffff0000u))) <= kMost4);
        if (bounded) {
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (no_number(v_two[g])) k_two[0] = 0x7fc07fc0u;
            store_values<true, __nv_bfloat16, G>(v, v_two, v_out + to, kMost4);
        } else {
            store_values<false, __nv_bfloat16, G>(v, v_two, v_out + to, 0.0f);
        }
        store_values<false, __nv_bfloat16, G>(k, k_two, k_out + to, 0.0f);
    }
}

template <typename T>
int launch_write(const void* qkv, void* q_out, const Pool4& k, const Pool4& v, const int* slots, const float* cos_t, const float* sin_t, const float* qw, const float* kw,
                 double eps, int n, int Hq, int Hkv, int D, int rotary, int page_size, int n_pages, cudaStream_t stream) {
    constexpr int kWarps = 4;
    const dim3 grid(n, (Hq + 2 * Hkv + kWarps - 1) / kWarps);
    const size_t smem = (size_t)kWarps * D * sizeof(double);
    const bool whole = rotary == 0 || rotary == D, aligned = (((size_t)cos_t | (size_t)sin_t | (size_t)qw | (size_t)kw) & 15) == 0;
    if ((D == 64 || D == 128 || D == 256) && whole && aligned) {
        auto lanes = D == 64 ? write_lanes_4bit_kernel<T, 2> : D == 128 ? write_lanes_4bit_kernel<T, 4> : write_lanes_4bit_kernel<T, 8>;
        const int heads = 128 / (D / 8), sections = (Hq + heads - 1) / heads + 2 * ((Hkv + heads - 1) / heads);
        return launch_pdl(lanes, dim3(n, sections), dim3(128), 0, stream, (const T*)qkv, (T*)q_out, k, v, slots, cos_t, sin_t, qw, kw, eps, Hq, Hkv,
                          rotary > 0 ? 1 : 0, page_size, n_pages, pool_bounds_now());
    }
    auto kernel = D <= 128 ? qk_norm_rope_write_4bit_kernel<T, 1> : qk_norm_rope_write_4bit_kernel<T, 2>;
    return launch_pdl(kernel, grid, dim3(kWarps * 32), smem, stream, (const T*)qkv, (T*)q_out, k, v, slots, cos_t, sin_t, qw, kw, eps, Hq, Hkv, D, rotary, page_size,
                      n_pages, pool_bounds_now());
}

// Arguments of an expansion; cu_q (and window): for attention.
struct Expand4 {
    Pool4 k, v;
    const int *table, *kv_len, *cu_q;
    void *k_out, *v_out;
    int* table_out;
    int n_seqs, width, Hkv, page_size, n_pages, window;
};
template <typename T, int G> int launch_expand_of(const Expand4& x, cudaStream_t stream) {
    const int units = 2 * x.Hkv * x.page_size * 4, blocks = (units + 511) / 512;         // two units a thread
    const dim3 grid(x.width, x.n_seqs, blocks < 64 ? blocks : 64);
    if (x.cu_q == nullptr)
        return launch_pdl(expand_pages_4bit_kernel<T, G>, grid, dim3(256), 0, stream, x.k, x.v, x.table, x.kv_len, (T*)x.k_out, (T*)x.v_out, x.table_out, x.width, x.Hkv,
                          x.page_size, x.n_pages, pool_bounds_now());
    if constexpr (sizeof(T) == 2 && (G == 2 || G == 4))                                  // what the dense kernels take
        return launch_pdl(expand_for_attention_4bit_kernel<G>, grid, dim3(256), 0, stream, x.k, x.v, x.table, x.kv_len, (T*)x.k_out, (T*)x.v_out, x.table_out, x.width, x.Hkv,
                          x.page_size, x.n_pages, x.cu_q, x.window, pool_bounds_now());
    return PB_ERR_BAD_SIZE;
}
template <typename T> int launch_expand(int groups, const Expand4& x, cudaStream_t stream) {
    switch (groups) {
#define PB_EXPAND(g) case g: return launch_expand_of<T, g>(x, stream);
        PB_EXPAND(1) PB_EXPAND(2) PB_EXPAND(3) PB_EXPAND(4) PB_EXPAND(5) PB_EXPAND(6) PB_EXPAND(7) PB_EXPAND(8)
#undef PB_EXPAND
    }
    return PB_ERR_BAD_SIZE;
}

bool sizes_4bit(int Hkv, int D, int page_size, int n_pages) {
    return Hkv > 0 && page_size > 0 && n_pages > 0 && D > 0 && D <= 256 && D % kGroup4 == 0;
}

}  // namespace

// dtype, qkv, q_out, k codes, k steps, v codes, v steps, slots, cos, sin, q weight, k weight, eps, n, Hq, Hkv, D, rotary, page_size, n_pages
PB_EXPORT int pb_qk_norm_rope_write_4bit(const long long* words, cudaStream_t stream) {
    Words4 w{words};
    const int dtype = w.num();
    const void* qkv = w.ptr<const void>();
    void* q_out = w.ptr<void>();
    Pool4 k, v;
    k.codes = w.ptr<uint8_t>();
    k.steps = w.ptr<__nv_bfloat16>();
    v.codes = w.ptr<uint8_t>();
    v.steps = w.ptr<__nv_bfloat16>();
    const int* slots = w.ptr<const int>();
    const float *cos_t = w.ptr<const float>(), *sin_t = w.ptr<const float>(), *q_weight = w.ptr<const float>(), *k_weight = w.ptr<const float>();
    const double eps = w.real();
    const int n = w.num(), Hq = w.num(), Hkv = w.num(), D = w.num(), rotary = w.num(), page_size = w.num(), n_pages = w.num();
    if (!sizes_4bit(Hkv, D, page_size, n_pages) || Hq < 0 || n < 0 || rotary < 0 || rotary > D || rotary % 2) return PB_ERR_BAD_SIZE;
    if (Hq + 2LL * Hkv > 65535) return PB_ERR_TOO_LARGE;
    if (n == 0) return 0;
    if (dtype == PB_F32)
        return launch_write<float>(qkv, q_out, k, v, slots, cos_t, sin_t, q_weight, k_weight, eps, n, Hq, Hkv, D, rotary, page_size, n_pages, stream);
    if (dtype == PB_BF16)
        return launch_write<__nv_bfloat16>(qkv, q_out, k, v, slots, cos_t, sin_t, q_weight, k_weight, eps, n, Hq, Hkv, D, rotary, page_size, n_pages, stream);
    return PB_ERR_BAD_DTYPE;
}

// dtype, k codes, k steps, v codes, v steps, table, kv_len, k out, v out, table out, n_seqs, width, Hkv, D, page_size, n_pages, cu_q (or 0), window
PB_EXPORT int pb_expand_pages_4bit(const long long* words, cudaStream_t stream) {
    Words4 w{words};
    const int dtype = w.num();
    Expand4 x;
    x.k.codes = w.ptr<uint8_t>();
    x.k.steps = w.ptr<__nv_bfloat16>();
    x.v.codes = w.ptr<uint8_t>();
    x.v.steps = w.ptr<__nv_bfloat16>();
    x.table = w.ptr<const int>();
    x.kv_len = w.ptr<const int>();
    x.k_out = w.ptr<void>();
    x.v_out = w.ptr<void>();
    x.table_out = w.ptr<int>();
    x.n_seqs = w.num();
    x.width = w.num();
    x.Hkv = w.num();
    const int D = w.num();
    x.page_size = w.num();
    x.n_pages = w.num();
    x.cu_q = w.ptr<const int>();
    x.window = w.num();
    if (!sizes_4bit(x.Hkv, D, x.page_size, x.n_pages) || x.n_seqs < 0 || x.width < 0 || x.window < 0) return PB_ERR_BAD_SIZE;
    if (x.n_seqs > 65535 || (long long)x.n_seqs * x.width > 0x7fffffffLL || (long long)x.width * x.page_size > 0x7fffffffLL || 8LL * x.Hkv * x.page_size > 0x3fffffffLL)
        return PB_ERR_TOO_LARGE;
    if (x.n_seqs == 0 || x.width == 0) return 0;
    if (dtype == PB_F32) return launch_expand<float>(D / kGroup4, x, stream);
    if (dtype == PB_BF16) return launch_expand<__nv_bfloat16>(D / kGroup4, x, stream);
    return PB_ERR_BAD_DTYPE;
}
