// Attention over keys and values held in 4 bits (cache4.cuh has the format).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  over the keys j that a query at position p sees: j <= p, and j > p - window
//
// A query token at place t of the n that its sequence brings stands at position kv_len - n + t; with cu_q null every sequence brings one.
// Keys whose page is not one of the pool are not seen.  A query that sees nothing gives zeros.
#include "cache4.cuh"

namespace {

using namespace pb;

// A block takes one query token and head, its warps every fourth run of 32 keys: a lane first scores a key, then gathers its channels of all 32 values.
template <typename T>
__global__ void paged_attention_4bit_kernel(const T* __restrict__ q, Pool4 k_pool, Pool4 v_pool, T* __restrict__ out, const int* __restrict__ table, int width,
                                            const int* __restrict__ kv_len, const int* __restrict__ cu_q, int n_seqs, int Hq, int Hkv, int D, int page_size, int n_pages,
                                            float scale, int window, const PoolBounds bounds) {
    pdl_wait();
    __shared__ float q_row[256], merged[4][256 + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x, head = blockIdx.y, G = D / kGroup4;
    int seq = row, pos = 0;
    if (cu_q == nullptr) {
        pos = kv_len[row] - 1;
    } else {
        if (row >= cu_q[n_seqs]) return;
        int low = 0, high = n_seqs;                    // cu_q[low] <= row < cu_q[high]
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if (cu_q[mid] <= row) low = mid; else high = mid;
        }
        seq = low;
        pos = kv_len[seq] - (cu_q[seq + 1] - row);
    }
    for (int i = threadIdx.x; i < D; i += blockDim.x) q_row[i] = to_float(q[((size_t)row * Hq + head) * D + i]) * scale;
    __syncthreads();
    const int first = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0, kvh = head / (Hq / Hkv);
    float most = -3.0e38f, total = 0.0f, o[2][4] = {};
    for (int at = first / 32 * 32 + 32 * warp; at <= pos; at += 128) {
        const int key = at + lane;
        size_t in_pool = 0;
        float score = -INFINITY;
        if (key >= first && key <= pos && key / page_size < width) {
            const int page = table[(size_t)seq * width + key / page_size];
            page_ok(page, bounds);
            if (page_or_none(page, n_pages) >= 0) {
                in_pool = ((size_t)page * Hkv + kvh) * page_size + key % page_size;
                score = 0.0f;
                for (int g = 0; g < G; ++g) {
                    const uint32_t two = reinterpret_cast<const uint32_t*>(k_pool.steps)[in_pool * G + g];
                    const float step = __uint_as_float(two << 16), least = __uint_as_float(two & 0xffff0000u);
                    for (int r = 0; r < 8; ++r) {
                        const uint32_t word = reinterpret_cast<const uint16_t*>(k_pool.codes)[in_pool * (size_t)(8 * G) + r * G + g];
                        for (int e = 0; e < 4; ++e) score = fmaf(q_row[32 * g + 4 * r + e], fmaf(step, (float)((word >> (4 * e)) & 15), least), score);
                    }
                }
            }
        }
        const bool seen = score != -INFINITY;
        const float now = fmaxf(most, warp_max(score));
        const float shrink = expf(most - now), p = seen ? expf(score - now) : 0.0f;
        most = now;
        total = total * shrink + p;
        for (int j = 0; j < 2; ++j) for (int e = 0; e < 4; ++e) o[j][e] *= shrink;
        for (int i = 0; i < 32; ++i) {
            const float w = __shfl_sync(0xffffffffu, p, i);
            const size_t there = __shfl_sync(0xffffffffu, in_pool, i);
            if (!__shfl_sync(0xffffffffu, (int)seen, i)) continue;
            for (int j = 0; j < 2; ++j) {
                const int quad = lane + 32 * j, g = quad >> 3, r = quad & 7;
                if (4 * quad >= D) break;
                const uint32_t two = reinterpret_cast<const uint32_t*>(v_pool.steps)[there * G + g];
                const float step = __uint_as_float(two << 16), least = __uint_as_float(two & 0xffff0000u);
                const uint32_t word = reinterpret_cast<const uint16_t*>(v_pool.codes)[there * (size_t)(8 * G) + r * G + g];
                for (int e = 0; e < 4; ++e) o[j][e] = fmaf(w, fmaf(step, (float)((word >> (4 * e)) & 15), least), o[j][e]);
            }
        }
    }
    total = warp_sum(total);
    for (int j = 0; j < 2; ++j) for (int e = 0; e < 4; ++e) if (4 * (lane + 32 * j) < D) merged[warp][4 * (lane + 32 * j) + e] = o[j][e];
    if (lane == 0) { merged[warp][256] = most; merged[warp][257] = total; }
    __syncthreads();
    float all = merged[0][256], below = 0.0f;
    for (int w = 1; w < 4; ++w) all = fmaxf(all, merged[w][256]);
    for (int w = 0; w < 4; ++w) below += expf(merged[w][256] - all) * merged[w][257];
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        float above = 0.0f;
        for (int w = 0; w < 4; ++w) above += expf(merged[w][256] - all) * merged[w][i];
        out[((size_t)row * Hq + head) * D + i] = from_float<T>(below == 0.0f ? 0.0f : above / below);
    }
}

}  // namespace

PB_EXPORT int pb_paged_attention_4bit(int dtype, const void* q, void* k_codes, void* k_steps, void* v_codes, void* v_steps, void* out, const int* table, int width,
                                      const int* kv_len, const int* cu_q, int n_rows, int n_seqs, int Hq, int Hkv, int D, int page_size, int n_pages, float scale,
                                      int window, cudaStream_t stream) {
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || D > 256 || D % kGroup4 || page_size <= 0 || n_pages <= 0 || width <= 0 || window < 0) return PB_ERR_BAD_SIZE;
    if (Hq > 65535) return PB_ERR_TOO_LARGE;
    if (n_rows == 0 || n_seqs == 0) return 0;
    const Pool4 k{(uint8_t*)k_codes, (__nv_bfloat16*)k_steps}, v{(uint8_t*)v_codes, (__nv_bfloat16*)v_steps};
    if (dtype == PB_F32)
        return launch_pdl(paged_attention_4bit_kernel<float>, dim3(n_rows, Hq), dim3(128), 0, stream, (const float*)q, k, v, (float*)out, table, width, kv_len, cu_q, n_seqs,
                          Hq, Hkv, D, page_size, n_pages, scale, window, pool_bounds_now());
    if (dtype == PB_BF16)
        return launch_pdl(paged_attention_4bit_kernel<__nv_bfloat16>, dim3(n_rows, Hq), dim3(128), 0, stream, (const __nv_bfloat16*)q, k, v, (__nv_bfloat16*)out, table,
                          width, kv_len, cu_q, n_seqs, Hq, Hkv, D, page_size, n_pages, scale, window, pool_bounds_now());
    return PB_ERR_BAD_DTYPE;
}
