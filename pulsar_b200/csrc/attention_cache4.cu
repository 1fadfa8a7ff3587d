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
// as the SMs hold at once, or as many as there are heads or least shares), or -n: a cluster of n blocks a head.  What ends first, by what was measured
// of heads of 128: with b blocks an SM a warp's turn takes 0.35 + 0.5 b us and a block's start and end 1 us more for each, and even shares 4 us for the
// second kernel and the look at all lengths.  (us, clusters of 1, 2, 4, 8 and even shares, 32 / 8 heads; sequences of half to all of so many keys:
// 1 of 900  9.0, 7.3, 6.2, 5.4, 9.9;  8 of 1,024  9.0, 7.8, 8.6, 12.5, 12.7;  8 of 4,096  26, 17.3, 14.8, 18.6, 17.4;  16 of 8,000  49, 36.3, 40, 42, 36.4;
// 64 of 1,024  23.6, 29, 39, 68, 30;  64 of 8,192  161, -, -, -, 106.)
PB_EXPORT int pb_attention_4bit_blocks(int dtype, int most_tokens, int n_seqs, int Hq, int Hkv, int D, int width, int page_size, int window) {
    if (Hkv <= 0 || Hq <= 0 || D <= 0 || most_tokens <= 0 || n_seqs <= 0 || width <= 0 || page_size <= 0) return 1;
    const int rows = pb_attention_4bit_rows(dtype, most_tokens * (Hq / Hkv), D), sms = sm_count_4bit(), held = blocks_4bit(dtype == PB_F32, D / kGroup4, rows);
    const long long row_blocks = ((long long)most_tokens * (Hq / Hkv) + rows - 1) / rows;
    long long keys = (long long)width * page_size;
    if (window > 0 && keys > (long long)window + most_tokens + 16) keys = (long long)window + most_tokens + 16;
    const long long heads = n_seqs * row_blocks * Hkv, of_head = (keys + kTile4 - 1) / kTile4, turns = heads * of_head, parts = (turns + kLeastShare4 - 1) / kLeastShare4;
    const int most = sms * held;
    if (row_blocks * Hkv <= 65535) {
        // in twentieths of a microsecond
        long long best = (turns + most * kWarps4 - 1) / (most * kWarps4) * (7 + 10 * held) + 20 * held + 80;
        int cluster = 0;
        for (int n = 1; n <= 8; n *= 2) {
            if (n > 1 && (heads * n > most || of_head < 3 * n)) continue;        // one wave of blocks, a turn for most of their warps
            const long long blocks = (heads * n + sms - 1) / sms, a_warp = (of_head + n * kWarps4 - 1) / (n * kWarps4);
            const long long takes = a_warp * (blocks <= held ? 7 + 10 * blocks : (7 + 10 * held) * blocks / held) + 20 * blocks;
            if (takes < best) {
                best = takes;
                cluster = n;
            }
        }
        if (cluster > 0) return -cluster;
    }
    const long long wanted = parts > heads ? parts : heads;
    return wanted < most ? (int)wanted : most;
}

namespace {
// Words: dtype, q, k codes, k steps, v codes, v steps, out, sums, plan, table, kv_len, cu_q (or 0), width, n_rows, most_tokens, n_seqs, Hq, Hkv, D, page_size,
// n_pages, scale, window, blocks (of attention_4bit_blocks; sums and plan only where it is above 0).
struct Call4 {
    Attend4 a;
    int dtype, D, most_tokens;
    double turns;                       // of all heads, at most
    // 0, or the error; `rows` of a block: 0 for attention_4bit_rows
    int read(const long long* words, int& rows) {
        Words4 w{words};
        dtype = w.num();
        a.q = w.ptr<const void>();
        a.k.codes = w.ptr<uint8_t>();
        a.k.steps = w.ptr<__nv_bfloat16>();
        a.v.codes = w.ptr<uint8_t>();
        a.v.steps = w.ptr<__nv_bfloat16>();
        a.out = w.ptr<void>();
        a.sums = w.ptr<float>();
        a.plan = w.ptr<int>();
        a.table = w.ptr<const int>();
        a.kv_len = w.ptr<const int>();
        a.cu_q = w.ptr<const int>();
        a.width = w.num();
        a.n_rows = w.num();
        most_tokens = w.num();
        a.n_seqs = w.num();
        a.Hq = w.num();
        a.Hkv = w.num();
        D = w.num();
        a.page_size = w.num();
        a.n_pages = w.num();
        a.scale_log2 = (float)w.real() * kLog2e;
        a.window = w.num();
        a.blocks = w.num();
        if (a.Hkv <= 0 || a.Hq <= 0 || a.Hq % a.Hkv || D <= 0 || D > 256 || D % kGroup4 || a.page_size <= 0 || a.n_pages <= 0 || a.width <= 0 || a.window < 0 || most_tokens < 0 ||
            a.n_seqs < 0 || a.n_rows < 0)
            return PB_ERR_BAD_SIZE;
        if (dtype != PB_F32 && dtype != PB_BF16) return PB_ERR_BAD_DTYPE;
        const int group = a.Hq / a.Hkv;
        if (rows == 0) rows = pb_attention_4bit_rows(dtype, most_tokens * group, D);
        const long long row_blocks = ((long long)most_tokens * group + rows - 1) / rows, keys = (long long)a.width * a.page_size;
        if (a.n_seqs > 65535 || (long long)most_tokens * a.Hq > 0x3fffffff || (long long)a.n_pages * a.Hkv * a.page_size >= 0xffffffffLL || keys > 0x7ffffff0LL) return PB_ERR_TOO_LARGE;
        turns = (double)a.n_seqs * row_blocks * a.Hkv * (keys / kTile4 + 1 + kGap4);
        a.page_shift = log2_exact(a.page_size);
        a.row_blocks = (int)row_blocks;
        a.bounds = pool_bounds_now();
        return 0;
    }
};
}  // namespace

PB_EXPORT int pb_paged_attention_4bit(const long long* words, cudaStream_t stream) {
    Call4 c;
    int rows = 0;
    if (const int rc = c.read(words, rows)) return rc;
    const Attend4& a = c.a;
    if (a.blocks == 0 || a.blocks < -8 || (a.blocks > 0 && (a.sums == nullptr || a.plan == nullptr))) return PB_ERR_BAD_SIZE;
    if (c.most_tokens == 0 || a.n_seqs == 0) return 0;
    if (c.turns > 1.0e9 || (a.blocks < 0 && (long long)a.row_blocks * a.Hkv > 65535)) return PB_ERR_TOO_LARGE;
    return (c.dtype == PB_F32 ? attend_4bit_f32 : attend_4bit_bf16)(a, c.D / kGroup4, rows, c.most_tokens, stream);
}

// Portions that a dense kernel has attended to over expanded pages: those that see keys of pages that are none.  Words as above, without sums, plan and
// blocks; bfloat16, heads of 64 or 128 (of which the dense kernels are).
PB_EXPORT int pb_paged_attention_4bit_holes(const long long* words, cudaStream_t stream) {
    Call4 c;
    int rows = 16;
    if (const int rc = c.read(words, rows)) return rc;
    if (c.dtype != PB_BF16 || c.a.cu_q == nullptr) return PB_ERR_BAD_DTYPE;
    if (c.most_tokens == 0 || c.a.n_seqs == 0) return 0;
    const bool by_16 = c.a.page_size % 16 == 0;
    const int sms = sm_count_4bit();
    if (c.D == 64) return by_16 ? launch_attend_4bit_holes<__nv_bfloat16, 2, 2, Turns16>(c.a, sms, stream) : launch_attend_4bit_holes<__nv_bfloat16, 2, 2, TurnsAny>(c.a, sms, stream);
    if (c.D == 128) return by_16 ? launch_attend_4bit_holes<__nv_bfloat16, 4, 2, Turns16>(c.a, sms, stream) : launch_attend_4bit_holes<__nv_bfloat16, 4, 2, TurnsAny>(c.a, sms, stream);
    return PB_ERR_BAD_SIZE;
}
