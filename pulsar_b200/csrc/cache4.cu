// Keys and values into a cache of 4 bits, and back (cache4.cuh has the format).
//
//   qk_norm_rope_write_4bit   per (token, head) of a projection row [q: Hq*D | k: Hkv*D | v: Hkv*D]: q and k are normed (x / sqrt(mean(x^2) + eps) * w,
//                             where weights are given) and their first `rotary` channels turned, (u, v) -> (u cos - v sin, v cos + u sin)
//                             with v half a turn's width behind u; q is rounded to T, k and v to T and then to 4 bits, at their slots.
//   expand_pages_4bit         the values of the pages that sequences hold, as T, into pages of their own.
#include "cache4.cuh"

namespace {

using namespace pb;

__device__ __forceinline__ float root_inverse(float v) { return rsqrtf(v); }
__device__ __forceinline__ double root_inverse(double v) { return 1.0 / sqrt(v); }
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
__device__ __forceinline__ void quantise_quad(const float (&y)[4], int quad, int groups, size_t at, const Pool4& pool) {
    float lo = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])), hi = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    constexpr float kMost = 3.38953139e38f;          // the largest bfloat16
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!(fabsf(y[e]) <= kMost)) hi = __int_as_float(0x7f800000);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (4 * quad >= kGroup4 * groups) return;
    const bool bad = hi > kMost;
    const double m = (double)__bfloat162float(__float2bfloat16_rd(lo));
    const float step = __bfloat162float(__float2bfloat16_ru(__double2float_ru(((double)hi - m) / 15.0)));
    const double s = (double)step, inverse = step > 0.0f ? 1.0 / s : 0.0;
    uint32_t word = 0;
    if (!bad) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double d = (double)y[e] - m;
            double c = d * inverse;
            c = fma(fma(-c, s, d), inverse, c);          // the quotient as a division would round it
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
    float y[QUADS][4];
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
    for (int j = 0; j < QUADS; ++j) quantise_quad(y[j], lane + 32 * j, D / kGroup4, at, is_k ? k_pool : v_pool);
}

// Eight channels of a row a thread: two words of codes and one of steps, 16 or 32 bytes of values.
template <typename T>
__global__ void expand_pages_4bit_kernel(Pool4 k_pool, Pool4 v_pool, const int* __restrict__ table, const int* __restrict__ kv_len, T* __restrict__ k_out,
                                         T* __restrict__ v_out, int* __restrict__ table_out, int width, int Hkv, int D, int page_size, int n_pages,
                                         const int* __restrict__ cu_q, int window, const PoolBounds bounds) {
    pdl_wait();
    const int seq = blockIdx.y, logical = blockIdx.x, length = kv_len[seq];
    const size_t out_page = (size_t)seq * width + logical;
    int rows = min(page_size, length - logical * page_size);                    // of this page, that hold a key
    int page = rows > 0 ? table[(size_t)seq * width + logical] : -1;
    if (rows > 0 && page >= 0) page_ok(page, bounds);
    bool there = page_or_none(page, n_pages) >= 0;
    if (cu_q != nullptr) {
        // For attention: what no tile of 128 keys that a query sees touches is left out, and what else is none becomes zeros.
        const int low = window > 0 ? length - (cu_q[seq + 1] - cu_q[seq]) - window + 1 - 128 : 0;
        if (!there) rows = min(rows, 0);
        there = logical * page_size < length && (logical + 1) * page_size > low;
    }
    if (blockIdx.z == 0 && threadIdx.x == 0) table_out[out_page] = there ? (int)out_page : -1;
    if (!there) return;
    const int G = D / kGroup4, octets = D / 8, per_head = page_size * octets, n = 2 * Hkv * per_head;
    for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < n; i += gridDim.z * blockDim.x) {
        const bool is_v = i >= Hkv * per_head;
        const int rest = is_v ? i - Hkv * per_head : i, row = rest / octets, o = rest - row * octets;      // row: head * page_size + place
        const Pool4& pool = is_v ? v_pool : k_pool;
        const int g = o >> 2, r = (o & 3) * 2;
        const size_t in_pool = (size_t)page * Hkv * page_size + row;
        float y[2][4] = {};
        if (row % page_size < rows) {
            const uint16_t* codes = reinterpret_cast<const uint16_t*>(pool.codes) + in_pool * (size_t)(8 * G);
            const uint32_t two = reinterpret_cast<const uint32_t*>(pool.steps)[in_pool * (size_t)G + g];
            const float step = __uint_as_float(two << 16), least = __uint_as_float(two & 0xffff0000u);
            const uint32_t words = codes[r * G + g] | (uint32_t)codes[(r + 1) * G + g] << 16;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e >> 2][e & 3] = fmaf(step, (float)((words >> (4 * e)) & 15), least);
        }
        T* dst = (is_v ? v_out : k_out) + (out_page * Hkv * page_size + row) * D + 8 * o;
        store_quad(dst, y[0]);
        store_quad(dst + 4, y[1]);
    }
}

template <typename T>
int launch_write(const void* qkv, void* q_out, const Pool4& k, const Pool4& v, const int* slots, const float* cos_t, const float* sin_t, const float* qw, const float* kw,
                 double eps, int n, int Hq, int Hkv, int D, int rotary, int page_size, int n_pages, cudaStream_t stream) {
    constexpr int kWarps = 4;
    const dim3 grid(n, (Hq + 2 * Hkv + kWarps - 1) / kWarps);
    const size_t smem = (size_t)kWarps * D * sizeof(double);
    auto kernel = D <= 128 ? qk_norm_rope_write_4bit_kernel<T, 1> : qk_norm_rope_write_4bit_kernel<T, 2>;
    return launch_pdl(kernel, grid, dim3(kWarps * 32), smem, stream, (const T*)qkv, (T*)q_out, k, v, slots, cos_t, sin_t, qw, kw, eps, Hq, Hkv, D, rotary, page_size,
                      n_pages, pool_bounds_now());
}

bool sizes_4bit(int Hkv, int D, int page_size, int n_pages) {
    return Hkv > 0 && page_size > 0 && n_pages > 0 && D > 0 && D <= 256 && D % kGroup4 == 0;
}

}  // namespace

PB_EXPORT int pb_qk_norm_rope_write_4bit(int dtype, const void* qkv, void* q_out, void* k_codes, void* k_steps, void* v_codes, void* v_steps, const int* slots,
                                         const float* cos_t, const float* sin_t, const float* q_weight, const float* k_weight, double eps, int n, int Hq, int Hkv, int D,
                                         int rotary, int page_size, int n_pages, cudaStream_t stream) {
    if (!sizes_4bit(Hkv, D, page_size, n_pages) || Hq < 0 || n < 0 || rotary < 0 || rotary > D || rotary % 2) return PB_ERR_BAD_SIZE;
    if ((Hq + 2 * Hkv + 3) / 4 > 65535) return PB_ERR_TOO_LARGE;
    if (n == 0) return 0;
    const Pool4 k{(uint8_t*)k_codes, (__nv_bfloat16*)k_steps}, v{(uint8_t*)v_codes, (__nv_bfloat16*)v_steps};
    if (dtype == PB_F32)
        return launch_write<float>(qkv, q_out, k, v, slots, cos_t, sin_t, q_weight, k_weight, eps, n, Hq, Hkv, D, rotary, page_size, n_pages, stream);
    if (dtype == PB_BF16)
        return launch_write<__nv_bfloat16>(qkv, q_out, k, v, slots, cos_t, sin_t, q_weight, k_weight, eps, n, Hq, Hkv, D, rotary, page_size, n_pages, stream);
    return PB_ERR_BAD_DTYPE;
}

PB_EXPORT int pb_expand_pages_4bit(int dtype, void* k_codes, void* k_steps, void* v_codes, void* v_steps, const int* table, const int* kv_len, void* k_out, void* v_out,
                                   int* table_out, int n_seqs, int width, int Hkv, int D, int page_size, int n_pages, const int* cu_q, int window,
                                   cudaStream_t stream) {
    if (!sizes_4bit(Hkv, D, page_size, n_pages) || n_seqs < 0 || width < 0 || window < 0) return PB_ERR_BAD_SIZE;
    if (n_seqs > 65535 || (long long)n_seqs * width > 0x7fffffffLL || 2LL * Hkv * page_size * (D / 8) > 0x3fffffffLL) return PB_ERR_TOO_LARGE;
    if (n_seqs == 0 || width == 0) return 0;
    const Pool4 k{(uint8_t*)k_codes, (__nv_bfloat16*)k_steps}, v{(uint8_t*)v_codes, (__nv_bfloat16*)v_steps};
    const int units = 2 * Hkv * page_size * (D / 8), blocks = (units + 1023) / 1024;
    const dim3 grid(width, n_seqs, blocks < 64 ? blocks : 64);
    if (dtype == PB_F32)
        return launch_pdl(expand_pages_4bit_kernel<float>, grid, dim3(256), 0, stream, k, v, table, kv_len, (float*)k_out, (float*)v_out, table_out, width, Hkv, D,
                          page_size, n_pages, cu_q, window, pool_bounds_now());
    if (dtype == PB_BF16)
        return launch_pdl(expand_pages_4bit_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, k, v, table, kv_len, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out,
                          table_out, width, Hkv, D, page_size, n_pages, cu_q, window, pool_bounds_now());
    return PB_ERR_BAD_DTYPE;
}
