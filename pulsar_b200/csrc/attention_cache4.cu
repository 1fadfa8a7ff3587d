// The bfloat16 kernels of attention over a cache of 4 bits (attention_cache4.cuh), and its entry point.
#include "attention_cache4.cuh"

namespace pb {

int attend_4bit_bf16(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream) {
    return launch_attend_4bit_of<__nv_bfloat16>(a, groups, rows, most_tokens, stream);
}

}  // namespace pb

using namespace pb;

// Rows that a block takes where a kv head has so many (its query heads times a sequence's tokens): 16 of bfloat16 heads of up to 128 where there are
// more than 8, for which registers suffice, 4 and 2 where there are no more and the head's groups of 32 channels can be dealt out to copies of them.
PB_EXPORT int pb_attention_4bit_rows(int dtype, int rows, int D) {
    if (rows > 8) return dtype == PB_BF16 && D <= 4 * kGroup4 ? 16 : 8;
    if (rows <= 2 && D % (4 * kGroup4) == 0) return 2;
    return rows <= 4 && D % (2 * kGroup4) == 0 ? 4 : 8;
}

namespace {
int sm_count_4bit() {
    static DeviceCount count;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    const int n = count.get(dev, [dev](int* v) { return (int)cudaDeviceGetAttribute(v, cudaDevAttrMultiProcessorCount, dev); });
    return n > 0 ? n : 148;
}
}  // namespace

// How a call is dealt out, by the longest sequences that the tables could name: n > 0 blocks in even shares whose parts a second kernel joins (as many
// as the SMs hold at once, or as many as there are heads or least shares), or -n: a cluster of n blocks a head.  The second kernel and
// the look at all lengths take some 4 us, which is what a block needs for kApart4 turns; clusters are taken where the fullest SM has no more
// turns than that above an even share.
constexpr int kApart4 = 25;
PB_EXPORT int pb_attention_4bit_blocks(int dtype, int most_tokens, int n_seqs, int Hq, int Hkv, int D, int width, int page_size, int window) {
    if (Hkv <= 0 || Hq <= 0 || D <= 0 || most_tokens <= 0 || n_seqs <= 0 || width <= 0 || page_size <= 0) return 1;
    const int rows = pb_attention_4bit_rows(dtype, most_tokens * (Hq / Hkv), D), sms = sm_count_4bit();
    const long long row_blocks = ((long long)most_tokens * (Hq / Hkv) + rows - 1) / rows;
    long long keys = (long long)width * page_size;
    if (window > 0 && keys > (long long)window + most_tokens + 16) keys = (long long)window + most_tokens + 16;
    const long long heads = n_seqs * row_blocks * Hkv, of_head = (keys + kTile4 - 1) / kTile4, turns = heads * of_head, parts = (turns + kLeastShare4 - 1) / kLeastShare4;
    const int most = sms * blocks_4bit(dtype == PB_F32, D / kGroup4, rows);
    if (row_blocks * Hkv <= 65535) {
        long long best = turns / sms + kApart4 + 1;
        int cluster = 0;
        for (int n = 8; n >= 1; n /= 2) {
            if (n > 1 && (heads * n > most || of_head < 3 * n)) continue;          // one wave of blocks, a turn for most of their warps
            const long long fullest = (heads * n + sms - 1) / sms * ((of_head + n - 1) / n);
            if (fullest < best) {
                best = fullest;
                cluster = n;
            }
        }
        if (cluster > 0) return -cluster;
    }
    const long long wanted = parts > heads ? parts : heads;
    return wanted < most ? (int)wanted : most;
}

// Words: dtype, q, k codes, k steps, v codes, v steps, out, sums, plan, table, kv_len, cu_q (or 0), width, n_rows, most_tokens, n_seqs, Hq, Hkv, D, page_size,
// n_pages, scale, window, blocks (of attention_4bit_blocks; sums and plan only where it is above 0).
PB_EXPORT int pb_paged_attention_4bit(const long long* words, cudaStream_t stream) {
    Words4 w{words};
    const int dtype = w.num();
    const void* q = w.ptr<const void>();
    Pool4 k, v;
    k.codes = w.ptr<uint8_t>();
    k.steps = w.ptr<__nv_bfloat16>();
    v.codes = w.ptr<uint8_t>();
    v.steps = w.ptr<__nv_bfloat16>();
    void* out = w.ptr<void>();
    float* sums = w.ptr<float>();
    int* plan = w.ptr<int>();
    const int *table = w.ptr<const int>(), *kv_len = w.ptr<const int>(), *cu_q = w.ptr<const int>();
    const int width = w.num(), n_rows = w.num(), most_tokens = w.num(), n_seqs = w.num(), Hq = w.num(), Hkv = w.num(), D = w.num(), page_size = w.num(), n_pages = w.num();
    const float scale = (float)w.real();
    const int window = w.num(), blocks = w.num();
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || D > 256 || D % kGroup4 || page_size <= 0 || n_pages <= 0 || width <= 0 || window < 0 || blocks == 0 || blocks < -8 ||
        (blocks > 0 && (sums == nullptr || plan == nullptr)) || most_tokens < 0 || n_seqs < 0 || n_rows < 0)
        return PB_ERR_BAD_SIZE;
    if (dtype != PB_F32 && dtype != PB_BF16) return PB_ERR_BAD_DTYPE;
    if (most_tokens == 0 || n_seqs == 0) return 0;
    const int group = Hq / Hkv, rows = pb_attention_4bit_rows(dtype, most_tokens * group, D);
    const long long row_blocks = ((long long)most_tokens * group + rows - 1) / rows, keys = (long long)width * page_size;
    if (n_seqs > 65535 || (long long)most_tokens * Hq > 0x3fffffff || (long long)n_pages * Hkv * page_size >= 0xffffffffLL || keys > 0x7ffffff0LL ||
        (double)n_seqs * row_blocks * Hkv * (keys / kTile4 + 1 + kGap4) > 1.0e9)
        return PB_ERR_TOO_LARGE;
    if (blocks < 0 && row_blocks * Hkv > 65535) return PB_ERR_TOO_LARGE;
    Attend4 a{q, out, k, v, sums, plan, table, kv_len, cu_q, width, n_rows, n_seqs,
              Hq, Hkv, page_size, log2_exact(page_size), n_pages, (int)row_blocks, blocks, window, scale * kLog2e, pool_bounds_now()};
    return (dtype == PB_F32 ? attend_4bit_f32 : attend_4bit_bf16)(a, D / kGroup4, rows, most_tokens, stream);
}
