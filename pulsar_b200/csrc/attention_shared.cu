// Decode attention over a forked cache: one query token per sequence, and families of sequences whose first keys lie in the same
// pages.  Those pages are read once for the family instead of once for each of its sequences.
//
// A softmax over keys cut into parts: with the part's maximum m_p, l_p = sum exp(s - m_p) and o_p = sum exp(s - m_p) v, the whole is
// o = sum_p exp(m_p - m) o_p / sum_p exp(m_p - m) l_p.  So the keys of a sequence are cut at shared_len: below it the query heads of ALL
// members of a family (members x group rows per kv head) meet each key tile together, above it each sequence's heads meet its own keys;
// both sides are cut further into splits, so that there are blocks enough, and a second kernel joins a row's parts.
//
// Bytes bound it: a key and a value of the shared part are read once per kv head and row tile, whatever the number of members.
//
// partial [n_seqs * Hq][n_shared + n_own][D + 2] float32: a part's o, then m (in units of log2) and l.
#include "mma_common.cuh"

namespace {

using namespace pb;

struct Shared {
    const int* block_table;
    const int* kv_len;          // [n_seqs]
    const int* shared_len;      // [n_seqs]: keys [0, shared_len) are read with the family; 0: no family
    const int* members;         // the families' sequences, one family behind the other
    const int* family_start;    // [n_families + 1]
    int n_seqs, n_members, n_families, most_members;
    int table_stride;
    int Hq, Hkv, page_size;
    int n_shared, n_own;        // splits of either side
    float scale_log2;
};

// What a block works on: keys [begin, end) read through `table`, and `rows` query rows from row `row0` of its family or sequence on.
struct Item {
    const int* table;
    int begin, end, rows, row0, first_member, seq, part;

    // row i of the item: its sequence and head
    __device__ __forceinline__ int seq_of(const Shared& p, int i, int G) const {
        return seq >= 0 ? seq : p.members[first_member + (row0 + i) / G];
    }
    __device__ __forceinline__ int head_of(int kvh, int i, int G) const { return kvh * G + (row0 + i) % G; }
};

// Blocks 0 .. n_families * family_tiles * n_shared - 1 are the shared sides', the rest the sequences' own.  False: nothing to do.
template <int ROWS, int TILE>
__device__ __forceinline__ bool item_of(const Shared& p, int block, int G, Item& it) {
    const int family_tiles = (p.most_members * G + ROWS - 1) / ROWS, own_tiles = (G + ROWS - 1) / ROWS;
    int keys, split, splits;
    const int shared_blocks = p.n_families * family_tiles * p.n_shared;
    if (block < shared_blocks) {
        split = block % p.n_shared;
        const int tile = block / p.n_shared % family_tiles, family = block / p.n_shared / family_tiles;
        it.first_member = p.family_start[family];
        const int count = min(min(p.family_start[family + 1], p.n_members) - it.first_member, p.most_members);
        if (it.first_member < 0 || count <= 0) return false;
        it.row0 = tile * ROWS;
        it.rows = min(ROWS, count * G - it.row0);
        if (it.rows <= 0) return false;
        const int first = p.members[it.first_member];
        if (first < 0 || first >= p.n_seqs) return false;
        it.table = p.block_table + (size_t)first * p.table_stride;
        it.begin = 0;
        keys = p.shared_len[first];
        it.seq = -1;
        it.part = split;
        splits = p.n_shared;
    } else {
        block -= shared_blocks;
        split = block % p.n_own;
        it.seq = block / p.n_own / own_tiles;
        it.row0 = block / p.n_own % own_tiles * ROWS;
        it.rows = min(ROWS, G - it.row0);
        it.first_member = 0;
        it.table = p.block_table + (size_t)it.seq * p.table_stride;
        it.begin = p.shared_len[it.seq];
        keys = p.kv_len[it.seq] - it.begin;
        it.part = p.n_shared + split;
        splits = p.n_own;
    }
    keys = max(0, min(keys, p.table_stride * p.page_size - it.begin));          // never beyond the table
    int chunk = (keys + splits - 1) / splits;
    chunk = (chunk + TILE - 1) / TILE * TILE;
    const int end = it.begin + keys;
    it.begin = min(end, it.begin + split * chunk);
    it.end = min(end, it.begin + chunk);
    return true;
}

// ---------------------------------------------------------------------------------------------
// Any head size that is a multiple of 16 (up to 256), any page size, float32 or bfloat16, on the CUDA cores in float32.  Four warps take
// four rows each of a tile of 16; a tile of 32 keys and its values are brought to shared memory as float32.  Scores: a lane per key; values:
// a lane per four of the head's dimensions.
constexpr int kRows = 16, kKeys = 32, kThreads = 128;
constexpr int kWarpRows = kRows / (kThreads / 32);

template <typename T, int QUADS /* groups of 128 dimensions */>
__global__ void __launch_bounds__(kThreads)
shared_general_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, float* __restrict__ partial,
                      const Shared p, int D, const PoolBounds bounds) {
    extern __shared__ __align__(16) float smem[];
    const int row_floats = D + 4;                        // 16-byte reads of 32 neighbouring rows then meet no bank twice
    float* q_s = smem;                                   // [kRows][D]
    float* k_s = q_s + kRows * D;                        // [kKeys][row_floats]
    float* v_s = k_s + kKeys * row_floats;               // [kKeys][D]
    const int kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = p.Hq / p.Hkv;
    Item it;
    if (!item_of<kRows, kKeys>(p, blockIdx.x, G, it)) return;
    const int quads = D / 4;
    for (int i = tid; i < kRows * quads; i += kThreads) {
        const int r = i / quads, d = (i - r * quads) * 4;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < it.rows) {
            const int seq = it.seq_of(p, r, G);
            if (seq >= 0 && seq < p.n_seqs) load_quad(q + ((size_t)seq * p.Hq + it.head_of(kvh, r, G)) * D + d, v);
        }
        store_quad(q_s + r * D + d, v);
    }
    float m[kWarpRows], l[kWarpRows], o[kWarpRows][QUADS][4];
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < QUADS; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.0f;
    }
    const int row0 = warp * kWarpRows;
    for (int key0 = it.begin; key0 < it.end; key0 += kKeys) {
        __syncthreads();
        for (int i = tid; i < kKeys * quads; i += kThreads) {
            const int r = i / quads, d = (i - r * quads) * 4, key = key0 + r;
            float kv[4] = {0.0f, 0.0f, 0.0f, 0.0f}, vv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (key < it.end) {
                int page = it.table[key / p.page_size];
                if (!page_ok(page, bounds)) page = 0;
                const size_t at = (((size_t)page * p.Hkv + kvh) * p.page_size + key % p.page_size) * D + d;
                load_quad(k_pool + at, kv);
                load_quad(v_pool + at, vv);
            }
            store_quad(k_s + r * row_floats + d, kv);
            store_quad(v_s + r * D + d, vv);
        }
        __syncthreads();
        if (row0 >= it.rows) continue;
        float s[kWarpRows];
#pragma unroll
        for (int r = 0; r < kWarpRows; ++r) s[r] = 0.0f;
        for (int d = 0; d < D; d += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(k_s + lane * row_floats + d);
#pragma unroll
            for (int r = 0; r < kWarpRows; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(q_s + (row0 + r) * D + d);
                s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
            }
        }
        const bool in = key0 + lane < it.end;
#pragma unroll
        for (int r = 0; r < kWarpRows; ++r) {
            s[r] = in ? s[r] * p.scale_log2 : -INFINITY;
            const float m_new = fmaxf(m[r], warp_max(s[r]));
            const float base = m_new == -INFINITY ? 0.0f : m_new;             // scores of -inf alone weigh nothing
            const float f = exp2f(m[r] - base);
            s[r] = exp2f(s[r] - base);
            l[r] = l[r] * f + s[r];
            m[r] = m_new;
#pragma unroll
            for (int j = 0; j < QUADS; ++j) { o[r][j][0] *= f; o[r][j][1] *= f; o[r][j][2] *= f; o[r][j][3] *= f; }
        }
        const int n = min(kKeys, it.end - key0);
        for (int key = 0; key < n; ++key) {
            float w[kWarpRows];
#pragma unroll
            for (int r = 0; r < kWarpRows; ++r) w[r] = __shfl_sync(0xffffffffu, s[r], key);
#pragma unroll
            for (int j = 0; j < QUADS; ++j) {
                const int d = (lane + 32 * j) * 4;
                if (d < D) {
                    const float4 v4 = *reinterpret_cast<const float4*>(v_s + key * D + d);
#pragma unroll
                    for (int r = 0; r < kWarpRows; ++r) {
                        o[r][j][0] = fmaf(w[r], v4.x, o[r][j][0]);
                        o[r][j][1] = fmaf(w[r], v4.y, o[r][j][1]);
                        o[r][j][2] = fmaf(w[r], v4.z, o[r][j][2]);
                        o[r][j][3] = fmaf(w[r], v4.w, o[r][j][3]);
                    }
                }
            }
        }
    }
    const int stride = D + 2, parts = p.n_shared + p.n_own;
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
        if (row0 + r >= it.rows) break;
        const int seq = it.seq_of(p, row0 + r, G);
        if (seq < 0 || seq >= p.n_seqs) continue;
        float* dst = partial + (((size_t)seq * p.Hq + it.head_of(kvh, row0 + r, G)) * parts + it.part) * stride;
        const float sum = warp_sum(l[r]);
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const int d = (lane + 32 * j) * 4;
            if (d < D) {
                dst[d] = o[r][j][0]; dst[d + 1] = o[r][j][1]; dst[d + 2] = o[r][j][2]; dst[d + 3] = o[r][j][3];
            }
        }
        if (lane == 0) { dst[D] = m[r]; dst[D + 1] = sum; }
    }
}

// Joins a row's parts: a warp per row.  A sequence outside the families has no shared parts.
template <typename T>
__global__ void __launch_bounds__(kThreads)
shared_join_kernel(const float* __restrict__ partial, T* __restrict__ out, const int* __restrict__ shared_len, int rows, int Hq, int D, int n_shared,
                   int n_own) {
    const int row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    const int parts = n_shared + n_own, stride = D + 2;
    const int first = shared_len[row / Hq] > 0 ? 0 : n_shared;
    const float* base = partial + (size_t)row * parts * stride;
    float m = -INFINITY;
    for (int i = first; i < parts; ++i) m = fmaxf(m, base[i * stride + D]);
    if (m == -INFINITY) m = 0.0f;                        // nothing to attend to (or NaN, which l carries)
    float l = 0.0f;
    for (int i = first; i < parts; ++i) l += base[i * stride + D + 1] * exp2f(base[i * stride + D] - m);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;       // a sequence without keys: zeros
    for (int d = lane; d < D; d += 32) {
        float acc = 0.0f;
        for (int i = first; i < parts; ++i) acc = fmaf(base[i * stride + d], exp2f(base[i * stride + D] - m), acc);
        out[(size_t)row * D + d] = from_float<T>(acc * inv);
    }
}

template <typename T>
int launch_general(const void* q, const void* k_pool, const void* v_pool, float* partial, const Shared& p, int D, int G, cudaStream_t stream) {
    const long long blocks = (long long)p.n_families * ((p.most_members * G + kRows - 1) / kRows) * p.n_shared +
                             (long long)p.n_seqs * ((G + kRows - 1) / kRows) * p.n_own;
    if (blocks > 0x7fffffff) return PB_ERR_TOO_LARGE;
    const size_t smem = (size_t)(kRows * D + kKeys * (D + 4) + kKeys * D) * sizeof(float);
    const dim3 grid((unsigned)blocks, p.Hkv);
    if (D <= 128) {
        static SmemLimit limit;
        if (const int rc = limit.allow(shared_general_kernel<T, 1>, smem)) return rc;
        shared_general_kernel<T, 1><<<grid, kThreads, smem, stream>>>((const T*)q, (const T*)k_pool, (const T*)v_pool, partial, p, D, pool_bounds_now());
    } else {
        static SmemLimit limit;
        if (const int rc = limit.allow(shared_general_kernel<T, 2>, smem)) return rc;
        shared_general_kernel<T, 2><<<grid, kThreads, smem, stream>>>((const T*)q, (const T*)k_pool, (const T*)v_pool, partial, p, D, pool_bounds_now());
    }
    return launch_status();
}

}  // namespace

// q, out [n_seqs, Hq, D], pools [pages, Hkv, page_size, D] (dtype 0 float32, 1 bfloat16); block_table int32 [n_seqs, table_stride];
// kv_len, shared_len int32 [n_seqs]; members int32 [n_members], family_start int32 [n_families + 1]; partial float32
// [n_seqs * Hq * (n_shared + n_own) * (D + 2)].
PB_EXPORT int pb_paged_attention_shared(int dtype, const void* q, const void* k_pool, const void* v_pool, void* out, float* partial,
                                        const int* block_table, int table_stride, const int* kv_len, const int* shared_len, const int* members,
                                        const int* family_start, int n_seqs, int n_members, int n_families, int most_members, int Hq, int Hkv, int D,
                                        int page_size, float scale, int n_shared, int n_own, cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (dtype != PB_F32 && dtype != PB_BF16) return PB_ERR_BAD_DTYPE;
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || D % 16 || D > 256 || page_size <= 0 || table_stride <= 0) return PB_ERR_BAD_SIZE;
    if (n_families < 0 || most_members < 0 || n_members < 0 || n_own <= 0 || n_shared < 0 || (n_families > 0 && n_shared == 0)) return PB_ERR_BAD_SIZE;
    if (Hkv > 65535 || n_shared + n_own > 256 || (long long)n_seqs * Hq > 0x7fffffff) return PB_ERR_TOO_LARGE;
    const int G = Hq / Hkv;
    Shared p{block_table, kv_len, shared_len, members, family_start, n_seqs, n_members, n_families, most_members, table_stride, Hq, Hkv, page_size, n_shared, n_own,
             scale * kLog2e};
    const int rc = dtype == PB_F32 ? launch_general<float>(q, k_pool, v_pool, partial, p, D, G, stream)
                                   : launch_general<bf16>(q, k_pool, v_pool, partial, p, D, G, stream);
    if (rc != 0) return rc;
    const int rows = n_seqs * Hq, blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
    if (dtype == PB_F32)
        shared_join_kernel<float><<<blocks, kThreads, 0, stream>>>(partial, (float*)out, shared_len, rows, Hq, D, n_shared, n_own);
    else
        shared_join_kernel<bf16><<<blocks, kThreads, 0, stream>>>(partial, (bf16*)out, shared_len, rows, Hq, D, n_shared, n_own);
    return launch_status();
}
