// What rows of logits say of given tokens: log probability, rank, the row's entropy and its likeliest tokens.
//
// One pass: every thread keeps the maximum and the sums (scores.cuh) of what it has seen.  The rank of the given token is a count of
// comparisons against its logit.
// The n likeliest (n <= 32) are kept by each warp as a list with one entry per lane, in order: a key of 64 bits holds the logit's
// bits, made to compare as unsigned numbers, above the complement of its index, so of equal logits the lower index is larger.  A
// logit enters only when it is beyond the list's last, which soon is rare.
// In the order of tokens a NaN is below every number.
#include "scores.cuh"

namespace {

using namespace pb;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
typedef unsigned long long Key;

__device__ __forceinline__ Key key_of(float x, int index) {
    const uint32_t bits = __float_as_uint(x + 0.0f);                          // -0 is +0
    const uint32_t up = x != x ? 0u : (bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u));
    return ((Key)up << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }

// Puts the warp's candidate (the same in all lanes, beyond the list's last) in its place.
__device__ __forceinline__ void insert(Key& list, Key candidate, int lane) {
    const int place = __popc(__ballot_sync(0xffffffffu, list > candidate));
    const Key above = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane >= place) list = lane == place ? candidate : above;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_scores_kernel(const T* __restrict__ logits, long long row_stride, int vocab, const int* __restrict__ tokens, float* __restrict__ logprob,
                    float* __restrict__ entropy, int* __restrict__ rank, int* __restrict__ top_ids, float* __restrict__ top_logprob, int n_top) {
    __shared__ Stats stats_s[kWarps];
    __shared__ int count_s[kWarps];
    __shared__ Key keys_s[kWarps * 32];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* row = logits + (long long)r * row_stride;
    const int token = tokens[r];
    const bool known = token >= 0 && token < vocab;
    const float given = known ? to_float(row[token]) : 0.0f;

    Stats st = {-INFINITY, 0.0f, 0.0f};
    int likelier = 0;
    Key list = 0, last = 0;
    for (int base = warp * 32; base < vocab; base += kThreads) {
        const int i = base + lane;
        const bool in = i < vocab;
        const float x = in ? to_float(row[i]) : -INFINITY;
        if (in) {
            if (x > st.m) {
                if (st.m > -INFINITY) {
                    const float delta = fmaxf(st.m - x, kFar), f = exp2f(delta * kScoreLog2e);
                    st.t = f * (st.t + st.s * delta);
                    st.s *= f;
                }
                st.m = x;
            }
            const float d = x - (st.m == -INFINITY ? 0.0f : st.m);
            const float e = exp2f(d * kScoreLog2e);
            st.s += e;
            st.t += e * fmaxf(d, kFar);
            likelier += (x > given || (x == given && i < token)) ? 1 : 0;
        }
        if (n_top > 0) {
            const Key key = in ? key_of(x, i) : 0;
            unsigned beyond = __ballot_sync(0xffffffffu, key > last);
            while (beyond) {
                const Key candidate = __shfl_sync(0xffffffffu, key, __ffs(beyond) - 1);
                insert(list, candidate, lane);
                last = __shfl_sync(0xffffffffu, list, n_top - 1);
                beyond &= beyond - 1;
                beyond &= __ballot_sync(0xffffffffu, key > last);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stats other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
        st = join(st, other);
        likelier += __shfl_xor_sync(0xffffffffu, likelier, o);
    }
    if (lane == 0) { stats_s[warp] = st; count_s[warp] = likelier; }
    if (n_top > 0) keys_s[warp * 32 + lane] = lane < n_top ? list : 0;
    __syncthreads();
    st = stats_s[0];
    likelier = count_s[0];
    for (int w = 1; w < kWarps; ++w) {
        st = join(st, stats_s[w]);
        likelier += count_s[w];
    }
    const float log_s = logf(st.s);
    if (tid == 0) {
        logprob[r] = known ? (given - st.m) - log_s : nanf("");
        entropy[r] = log_s - st.t / st.s;
        if (rank != nullptr) rank[r] = known ? likelier : -1;
    }
    // a key's place among all warps' lists is the number of larger ones (no two are equal but the empty ones, which are smallest)
    for (int i = tid; i < kWarps * n_top; i += kThreads) {
        const Key key = keys_s[i / n_top * 32 + i % n_top];
        if (key == 0) continue;
        int place = 0;
        for (int w = 0; w < kWarps; ++w)
            for (int j = 0; j < n_top && keys_s[w * 32 + j] > key; ++j) ++place;
        if (place < n_top) {
            const int index = index_of(key);
            top_ids[(long long)r * n_top + place] = index;
            top_logprob[(long long)r * n_top + place] = (to_float(row[index]) - st.m) - log_s;
        }
    }
}

}  // namespace

// logits [rows, vocab] (dtype 0 float32, 1 bfloat16), row_stride elements from a row to the next; tokens, rank, top_ids int32, the other
// results float32; rank may be null, top_ids and top_logprob [rows, n_top] are null where n_top is 0 (n_top <= 32, <= vocab).
PB_EXPORT int pb_token_scores(int dtype, const void* logits, long row_stride, int rows, int vocab, const int* tokens, float* logprob, float* entropy,
                              int* rank, int* top_ids, float* top_logprob, int n_top, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || n_top < 0 || n_top > 32 || n_top > vocab || row_stride < 0) return PB_ERR_BAD_SIZE;
    if (n_top > 0 && (top_ids == nullptr || top_logprob == nullptr)) return PB_ERR_BAD_SIZE;
    if (dtype == PB_F32)
        token_scores_kernel<float><<<rows, kThreads, 0, stream>>>((const float*)logits, row_stride, vocab, tokens, logprob, entropy, rank, top_ids,
                                                                  top_logprob, n_top);
    else if (dtype == PB_BF16)
        token_scores_kernel<__nv_bfloat16><<<rows, kThreads, 0, stream>>>((const __nv_bfloat16*)logits, row_stride, vocab, tokens, logprob, entropy,
                                                                          rank, top_ids, top_logprob, n_top);
    else
        return PB_ERR_BAD_DTYPE;
    return launch_status();
}
