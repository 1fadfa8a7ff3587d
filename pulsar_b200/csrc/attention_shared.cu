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
#include "attention_shared.cuh"
#include "mma_common.cuh"
#include "tcgen05_common.cuh"

#include <type_traits>

namespace {

using namespace pb;

using namespace pb::shared_attention;

// ---------------------------------------------------------------------------------------------
// Any head size that is a multiple of 16 (up to 256), any page size, float32 or bfloat16, on the CUDA cores in float32.  16 rows meet tiles
// of 64 keys, of which each of four warps has 16, with a maximum, sums and an O of its own; the four are joined at the end.  A warp's scores
// are 16 rows x 16 keys, four rows and two keys a lane, its O 16 rows x D, four dimensions a lane: shared memory is then read 6 times per 32
// products of scores and 5 per 64 of O, and the shared sides are bound by these instructions; items of up to 4 or 8 rows (a sequence's own) leave out the
// rest and are bound by bytes.  Keys and values come by cp.async as they lie in the pools, the next tile's keys under this one's values and its
// values under the next one's scores.  (float32, heads of 128: 4 families of 8 over 2,000 keys 59 us, four times what the multiply-adds take at their units' rate, where a key a lane and four rows a
// warp, 5 reads per 16 products, took 156; 30 sequences of 2,000 keys that share nothing 82 us, 6.4 TB/s.)
constexpr int kRows = 16, kKeys = 64, kThreads = 128;
constexpr int kWarpKeys = kKeys / (kThreads / 32);
constexpr int kWeightPitch = 20;                         // floats from a key's 16 weights to the next key's: stored and read without bank conflicts

__device__ __forceinline__ void load_eight(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load_eight(const bf16* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

// Shared memory: queries, weights and factors, keys, values.  A row of queries or keys is 16 bytes longer than its elements, so that 8 rows of
// keys, or 4 of queries, are read without bank conflicts.
template <typename T> constexpr int kRowPad = 16 / (int)sizeof(T);
template <typename T>
size_t general_smem(int D) {
    return kRows * (D + 4) * sizeof(float) + (kKeys * kWeightPitch + kThreads / 32 * kRows) * sizeof(float) + kKeys * (2 * D + kRowPad<T>) * sizeof(T);
}

template <typename T, int QUADS /* groups of 128 dimensions */>
__global__ void __launch_bounds__(kThreads)
shared_general_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, float* __restrict__ partial,
                      const Shared p, int shared_blocks, int D, const PoolBounds bounds) {
    extern __shared__ __align__(16) float smem[];
    __shared__ long long row_s[2][kKeys];                // where in the pools the rows of a tile lie, -1: beyond the item's keys
    const int q_pitch = D + 4, k_pitch = D + kRowPad<T>;
    float* q_s = smem;                                   // [kRows][q_pitch]
    float* weight_s = q_s + kRows * q_pitch;             // [kKeys][kWeightPitch]
    float* factor_s = weight_s + kKeys * kWeightPitch;   // [warps][kRows]
    T* k_s = reinterpret_cast<T*>(factor_s + kThreads / 32 * kRows);         // [kKeys][k_pitch]
    T* v_s = k_s + kKeys * k_pitch;                      // [kKeys][D]
    const int kvh = blockIdx.x % p.Hkv, block = blockIdx.x / p.Hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = p.Hq / p.Hkv;
    Item it;
    pdl_trigger();                                       // (the join waits for this kernel's end)
    if (block >= shared_blocks ? !own_item<kRows>(p, block - shared_blocks, G, it) : !family_item<kRows, kKeys>(p, block, G, it)) return;
    auto row_of = [&](int key) {
        if (key >= it.end) return -1ll;
        int page = it.table[key / p.page_size];
        if (!page_ok(page, bounds)) page = 0;
        return (((long long)page * p.Hkv + kvh) * p.page_size + key % p.page_size) * D;
    };
    constexpr int kChunk = 16 / (int)sizeof(T);
    const int chunks = D / kChunk, first_row = tid / chunks, first_chunk = tid - first_row * chunks;
    const int row_step = kThreads / chunks, chunk_step = kThreads - row_step * chunks;
    auto fetch = [&](const T* pool, T* tile, int pitch, const long long* row) {              // rows beyond the item's keys become zeros
        for (int r = first_row, c = first_chunk; r < kKeys;) {
            const long long at = row[r];
            cp_async16(smem_addr(tile + r * pitch + c * kChunk), pool + (at < 0 ? 0 : at) + c * kChunk, at >= 0);
            r += row_step;
            c += chunk_step;
            if (c >= chunks) { c -= chunks; ++r; }
        }
        cp_async_commit();
    };
    if (tid < kKeys) {
        row_s[0][tid] = row_of(it.begin + tid);
        row_s[1][tid] = row_of(it.begin + kKeys + tid);
    }
    __syncthreads();
    if (it.begin < it.end) {
        fetch(k_pool, k_s, k_pitch, row_s[0]);
        fetch(v_pool, v_s, D, row_s[0]);
    }
    const int quads = D / 4;
    for (int i = tid; i < kRows * quads; i += kThreads) {
        const int r = i / quads, d = (i - r * quads) * 4;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < it.rows) {
            const int seq = it.seq_of(p, r, G);
            if (seq >= 0 && seq < p.n_seqs) load_quad(q + ((size_t)seq * p.Hq + it.head_of(kvh, r, G)) * D + d, v);
        }
        store_quad(q_s + r * q_pitch + d, v);
    }
    const int key_lane = lane & 7, row_lane = lane >> 3, key_warp = warp * kWarpKeys;        // rows row_lane + 4 i, keys key_lane and + 8
    float m[4], l[4], o[kRows][QUADS][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int j = 0; j < QUADS; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.0f;
    cp_async_wait<1>();
    __syncthreads();                                                          // the first keys, and the queries
    auto walk = [&](auto quarters) {                     // of the 16 rows: those that the item has
        constexpr int N = decltype(quarters)::value;
        int turn = 0;
        for (int key0 = it.begin; key0 < it.end; key0 += kKeys, ++turn) {
            const bool more = key0 + kKeys < it.end, mine = key0 + key_warp < it.end;
            const long long row_later = tid < kKeys ? row_of(key0 + 2 * kKeys + tid) : 0;
            bool moved = false;
            if (mine) {
                float s[4][2] = {};
                const T* key_a = k_s + (key_warp + key_lane) * k_pitch;
                const T* key_b = key_a + 8 * k_pitch;
                const float* query = q_s + row_lane * q_pitch;
#pragma unroll 2
                for (int d = 0; d < D; d += 8) {
                    float a[8], b[8];
                    load_eight(key_a + d, a);
                    load_eight(key_b + d, b);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float x[8];
                        load_eight(query + 4 * i * q_pitch + d, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            s[i][0] = fmaf(x[e], a[e], s[i][0]);
                            s[i][1] = fmaf(x[e], b[e], s[i][1]);
                        }
                    }
                }
                const bool in_a = key0 + key_warp + key_lane < it.end, in_b = key0 + key_warp + key_lane + 8 < it.end;
                float* weight = weight_s + (key_warp + key_lane) * kWeightPitch + row_lane;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float a = in_a ? s[i][0] * p.scale_log2 : -INFINITY, b = in_b ? s[i][1] * p.scale_log2 : -INFINITY;
                    float top = fmaxf(a, b);
#pragma unroll
                    for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float m_new = fmaxf(m[i], top), base = m_new == -INFINITY ? 0.0f : m_new;      // scores of -inf alone weigh nothing
                    const float f = exp2f(m[i] - base), wa = exp2f(a - base), wb = exp2f(b - base);
                    l[i] = l[i] * f + (wa + wb);
                    m[i] = m_new;
                    weight[4 * i] = wa;
                    weight[4 * i + 8 * kWeightPitch] = wb;
                    if (key_lane == 0) factor_s[warp * kRows + row_lane + 4 * i] = f;
                    moved = moved || f != 1.0f;
                }
                moved = __any_sync(0xffffffffu, moved);
            }
            cp_async_wait<0>();
            __syncthreads();                                                      // this tile's values; all are done with its keys
            if (tid < kKeys) row_s[turn & 1][tid] = row_later;
            if (more) fetch(k_pool, k_s, k_pitch, row_s[(turn + 1) & 1]);
            if (mine) {
                if (moved) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float4 f4 = *reinterpret_cast<const float4*>(factor_s + warp * kRows + 4 * i);
                        const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int j = 0; j < QUADS; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[4 * i + r][j][e] *= f[r];
                    }
                }
                const float* weight = weight_s + key_warp * kWeightPitch;
                const T* value = v_s + key_warp * D + lane * 4;
#pragma unroll 2
                for (int key = 0; key < kWarpKeys; ++key) {                       // (weights beyond the item's keys are zeros, and so are the values)
                    float v[QUADS][4];
#pragma unroll
                    for (int j = 0; j < QUADS; ++j) {
                        v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.0f;
                        if ((lane + 32 * j) * 4 < D) load_quad(value + key * D + 128 * j, v[j]);
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float4 w4 = *reinterpret_cast<const float4*>(weight + key * kWeightPitch + 4 * i);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int j = 0; j < QUADS; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[4 * i + r][j][e] = fmaf(w[r], v[j][e], o[4 * i + r][j][e]);
                    }
                }
            }
            cp_async_wait<0>();
            __syncthreads();                                                      // the next tile's keys; all are done with this one's values
            if (more) fetch(v_pool, v_s, D, row_s[(turn + 1) & 1]);
        }
    };
    if (it.rows <= 4) walk(std::integral_constant<int, 1>());
    else if (it.rows <= 8) walk(std::integral_constant<int, 2>());
    else walk(std::integral_constant<int, 4>());
    // The four warps meet in the memory of keys and values (256 D bytes, which either type's tiles have).
    float* o_s = reinterpret_cast<float*>(k_s);                               // [warps][kRows][D]
    float2* ml_s = reinterpret_cast<float2*>(weight_s);                       // [warps][kRows]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        if (key_lane == 0) ml_s[warp * kRows + row_lane + 4 * i] = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
            if (r < it.rows && (lane + 32 * j) * 4 < D) store_quad(o_s + (warp * kRows + r) * D + (lane + 32 * j) * 4, o[r][j]);
    __syncthreads();
    const int stride = D + 2, parts = p.n_shared + p.n_own;
    for (int i = tid; i < it.rows * quads; i += kThreads) {
        const int r = i / quads, d = (i - r * quads) * 4, seq = it.seq_of(p, r, G);
        if (seq < 0 || seq >= p.n_seqs) continue;
        float top = -INFINITY, sum = 0.0f, acc[4] = {};
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, ml_s[w * kRows + r].x);
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            const float2 ml = ml_s[w * kRows + r];
            const float f = exp2f(ml.x - (top == -INFINITY ? 0.0f : top));
            float v[4];
            load_quad(o_s + (w * kRows + r) * D + d, v);
            sum = fmaf(ml.y, f, sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], f, acc[e]);
        }
        float* dst = partial + (((size_t)seq * p.Hq + it.head_of(kvh, r, G)) * parts + it.part) * stride;
        *reinterpret_cast<float2*>(dst + d) = make_float2(acc[0], acc[1]);
        *reinterpret_cast<float2*>(dst + d + 2) = make_float2(acc[2], acc[3]);
        if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(top, sum);
    }
}

// ---------------------------------------------------------------------------------------------
// bfloat16, head size 64 or 128, pages of 8, 16, 32 or 64 keys: on the tensor cores (mma.m16n8k16, float32 sums).  Tiles of 64 keys and
// values come page by page through TMA (boxes of a page x 64 dimensions, 128-byte swizzle) into a ring that a warp of its own fills,
// two or three blocks an SM: what limits the kernel is bytes in flight, and instructions that gather a tile would cost the other warps as
// much as its products (cp.async by all warps: 2,300 cycles a tile and block; 101 sequences, 96 of them in 12 families over up to 2,600
// keys: 77 against 66 us).  ROW_TILES x 16 query rows meet each tile; the four warps share the work as ROW_TILES row tiles x 4 / ROW_TILES
// parts of the tile's keys: with one row tile (a sequence's own keys) each warp has 16 keys, with four each has all 64 for its own rows, so
// that shared memory is read no more often than rows need.  (The 101 sequences' own keys, up to 500 each, 115 MB: 33 us cold, 44 % of the
// memory's rate: walks of a few tiles, which their starts and ends bound.)
//
// Rows of a tile that no key of the item fills hold what lies in the page, or an earlier tile: their scores are masked, and their values
// are overwritten with zeros, for zero weights do not silence a NaN.  Every wait is bounded; a block that gives up sets the error
// word, lets its copies land and returns.
constexpr int kTile = 64, kWarps = 4, kTcThreads = (kWarps + 1) * 32;
// Blocks of one row tile (a sequence's own keys: short walks, whose starts and ends others have to hide) run three to an SM, others two.
template <int ROW_TILES> constexpr int kBlocks = ROW_TILES == 1 ? 3 : 2;
template <int ROW_TILES> constexpr int kRing = (ROW_TILES == 1 ? 64 : 96) * 1024;
template <int D> constexpr int kTileBytes = kTile * D * 2;                    // of keys, and of values

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile: halves of 64 dimensions, rows of 128 bytes, swizzled as TMA leaves them.
__device__ __forceinline__ uint32_t tma_offset(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * (kTile * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

struct Ring {
    uint64_t full[8], empty[8];
    int gave_up;
};

// The warp that fills the ring, a lane per page of a tile.  False: a wait ran out.
template <int D, int STAGES>
__device__ __forceinline__ bool fill(const CUtensorMap* map_k, const CUtensorMap* map_v, const Shared& p, const Item& it, int kvh, int page_shift,
                                     const PoolBounds& bounds, uint32_t ring, Ring& sync) {
    const int lane = threadIdx.x & 31;
    int at = 0;
    for (int key0 = it.begin; key0 < it.end; key0 += kTile, ++at) {               // (an item begins with a page)
        const int stage = at % STAGES;
        const int first = key0 >> page_shift, last = (min(it.end, key0 + kTile) - 1) >> page_shift;      // pages of the tile
        int page = first + lane <= last ? it.table[first + lane] : 0;
        if (!page_ok(page, bounds)) page = 0;
        const uint32_t full = smem_addr(&sync.full[stage]);
        bool ok = true;
        if (lane == 0) {
            ok = mbar_wait(smem_addr(&sync.empty[stage]), ((at / STAGES) & 1) ^ 1, &sync.gave_up);
            if (ok) mbar_expect_tx(full, (uint32_t)((last - first + 1) << page_shift) * D * 4);
        }
        if (!__shfl_sync(0xffffffffu, (int)ok, 0)) return false;
        if (first + lane <= last) {
            const uint32_t dst = ring + stage * 2 * kTileBytes<D> + (lane << page_shift) * 128;
            const int row = (page * p.Hkv + kvh) << page_shift;
#pragma unroll
            for (int half = 0; half < D / 64; ++half) {
                tma_load_2d(dst + half * kTile * 128, map_k, full, half * 64, row);
                tma_load_2d(dst + kTileBytes<D> + half * kTile * 128, map_v, full, half * 64, row);
            }
        }
        __syncwarp();
    }
    return true;
}

// The four warps that compute meet here.
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// The warps that compute.  False: a wait ran out (the warps still meet).
template <int D, int ROW_TILES, int STAGES>
__device__ __forceinline__ bool attend(const bf16* __restrict__ q, float* __restrict__ partial, const Shared& p, const Item& it, int kvh, int G, uint32_t ring,
                                       unsigned char* smem, Ring& sync) {
    constexpr int kKSteps = D / 16, kNTiles = D / 8;
    constexpr int kKeyParts = kWarps / ROW_TILES, kGroups = ROW_TILES;           // groups of 16 keys that a warp has of a tile
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int row_tile = warp % ROW_TILES, key_part = warp / ROW_TILES;
    // the warp's query rows: row_tile * 16 + g and + 8, as sequence * Hq + head, or -1
    int rows[2];
    uint32_t qa[kKSteps][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = row_tile * 16 + g + 8 * r;
        rows[r] = -1;
        if (i < it.rows) {
            const int seq = it.seq_of(p, i, G);
            if (seq >= 0 && seq < p.n_seqs) rows[r] = seq * p.Hq + it.head_of(kvh, i, G);
        }
        const bf16* from = q + (size_t)max(rows[r], 0) * D + 2 * t;
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
            qa[ks][r] = rows[r] >= 0 ? *reinterpret_cast<const uint32_t*>(from + ks * 16) : 0u;
            qa[ks][r + 2] = rows[r] >= 0 ? *reinterpret_cast<const uint32_t*>(from + ks * 16 + 8) : 0u;
        }
    }
    float o[kNTiles][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kNTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const bool has_rows = row_tile * 16 < it.rows;
    bool ok = true;
    int at = 0;
    for (int tile0 = it.begin; tile0 < it.end; tile0 += kTile, ++at) {
        const int stage = at % STAGES;
        ok = mbar_wait(smem_addr(&sync.full[stage]), (at / STAGES) & 1, &sync.gave_up);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t k_s = ring + stage * 2 * kTileBytes<D>, v_s = k_s + kTileBytes<D>;
        const int in_tile = key_part * kGroups * 16, key0 = tile0 + in_tile;
        if (has_rows && key0 < it.end) {
            const bool inside = key0 + kGroups * 16 <= it.end;
            if (!inside) {
                // values of rows without a key become zeros (warps with the same rows write the same)
                for (int c = lane; c < kGroups * 16 * (D / 8); c += 32) {
                    const int row = c / (D / 8);
                    if (key0 + row >= it.end)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_s + tma_offset(in_tile + row, c % (D / 8))), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before TMA fills the stage again
                __syncwarp();
            }
            float s[2 * kGroups][4];
#pragma unroll
            for (int n = 0; n < 2 * kGroups; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < kKSteps; ++ks)
#pragma unroll
                for (int n = 0; n < kGroups; ++n) {
                    uint32_t kb[4];
                    ldmatrix_x4(kb, k_s + tma_offset(in_tile + n * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
                    mma_bf16(s[2 * n], qa[ks], kb[0], kb[1]);
                    mma_bf16(s[2 * n + 1], qa[ks], kb[2], kb[3]);
                }
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 2 * kGroups; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + n * 8 + 2 * t + (e & 1);
                    s[n][e] = inside || key < it.end ? s[n][e] * p.scale_log2 : -INFINITY;
                    top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
                }
            float f[2], base[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                const float m_new = fmaxf(m[r], top[r]);
                base[r] = m_new == -INFINITY ? 0.0f : m_new;                      // scores of -inf alone weigh nothing
                f[r] = pow2(m[r] - base[r]);
                m[r] = m_new;
                l[r] *= f[r];
            }
#pragma unroll
            for (int n = 0; n < 2 * kGroups; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = pow2(s[n][e] - base[e >> 1]);
                    l[e >> 1] += s[n][e];
                }
            if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {          // a maximum rose, which soon is rare
#pragma unroll
                for (int j = 0; j < kNTiles; ++j) { o[j][0] *= f[0]; o[j][1] *= f[0]; o[j][2] *= f[1]; o[j][3] *= f[1]; }
            }
#pragma unroll
            for (int n = 0; n < kGroups; ++n) {
                // weights in [0, 1], rounded to bfloat16 for the product (2^-9 of each, at random: 2.2e-3 of a result, 1.7e-3 of which are the
                // result's own rounding; float32 weights would take two products); their sum is of the unrounded ones
                const uint32_t pa[4] = {pack_bf16(s[2 * n][0], s[2 * n][1]), pack_bf16(s[2 * n][2], s[2 * n][3]),
                                        pack_bf16(s[2 * n + 1][0], s[2 * n + 1][1]), pack_bf16(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
                for (int j = 0; j < kNTiles; j += 2) {
                    uint32_t vb[4];
                    ldmatrix_x4_trans(vb, v_s + tma_offset(in_tile + n * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), j + (lane >> 4)));
                    mma_bf16(o[j], pa, vb[0], vb[1]);
                    mma_bf16(o[j + 1], pa, vb[2], vb[3]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sync.empty[stage]));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    const int stride = D + 2, parts = p.n_shared + p.n_own;
    if (kKeyParts == 1) {
        if (!ok) return false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (rows[r] < 0) continue;
            float* dst = partial + ((size_t)rows[r] * parts + it.part) * stride;
#pragma unroll
            for (int j = 0; j < kNTiles; ++j) *reinterpret_cast<float2*>(dst + j * 8 + 2 * t) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
            if (t == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[r], l[r]);
        }
        return true;
    }
    // The warps that had other keys of the same rows meet in shared memory: [row][key part][kPitch] floats of o, then m, l and the row's number.
    constexpr int kPitch = D + 8;                                                 // eight rows of a warp meet different banks
    float* merge = reinterpret_cast<float*>(smem);
    meet();                                                                       // all tiles have been read
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = row_tile * 16 + g + 8 * r;
        if (i < it.rows) {
            float* at_row = merge + (i * kKeyParts + key_part) * kPitch;
#pragma unroll
            for (int j = 0; j < kNTiles; ++j) *reinterpret_cast<float2*>(at_row + j * 8 + 2 * t) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
            if (t == 0) *reinterpret_cast<float4*>(at_row + D) = make_float4(m[r], l[r], __int_as_float(rows[r]), 0.0f);
        }
    }
    meet();
    if (!ok) return false;
    for (int i = tid; i < it.rows * (D / 4); i += kWarps * 32) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        const float* from = merge + row * kKeyParts * kPitch;
        const int to = __float_as_int(from[D + 2]);
        if (to < 0) continue;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kKeyParts; ++w) top = fmaxf(top, from[w * kPitch + D]);
        const float base = top == -INFINITY ? 0.0f : top;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kKeyParts; ++w) {
            const float f = pow2(from[w * kPitch + D] - base);
            const float4 v = *reinterpret_cast<const float4*>(from + w * kPitch + d);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
            sum = fmaf(from[w * kPitch + D + 1], f, sum);
        }
        float* dst = partial + ((size_t)to * parts + it.part) * stride;
        *reinterpret_cast<float2*>(dst + d) = make_float2(acc.x, acc.y);
        *reinterpret_cast<float2*>(dst + d + 2) = make_float2(acc.z, acc.w);
        if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(top, sum);
    }
    return true;
}

// ROW_TILES: of the shared sides' items; a sequence's own keys meet tiles of 16 rows.  Blocks in the order of the grid, the kv head fastest:
// the shared sides', then the first parts of all sequences' own keys, then their second, which many do not have.  (Blocks that walk over items
// and ask for the next one's tiles ahead were no faster, 75 against 57 us for the 101
// sequences above: the shares come out uneven.)  beside: the kernel
// before it on the stream has the shared sides; it was launched the ordinary way, lets this one in at its start, and the two write
// different parts.
template <int D, int ROW_TILES>
__global__ void __launch_bounds__(kTcThreads, kBlocks<ROW_TILES>)
shared_tc_kernel(const bf16* __restrict__ q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 float* __restrict__ partial, const Shared p, int shared_items, int page_shift, const PoolBounds bounds, unsigned int* error, bool beside) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ Ring sync;
    constexpr int kStages = kRing<ROW_TILES> / (2 * kTileBytes<D>);
    pdl_trigger();                                                                // (the join waits for this kernel's end)
    const int G = p.Hq / p.Hkv, tid = threadIdx.x, warp = tid >> 5, kvh = blockIdx.x % p.Hkv, block = blockIdx.x / p.Hkv;
    const bool family = block < shared_items;
    Item it;
    if (family ? family_item<ROW_TILES * 16, kTile>(p, block, G, it) : own_item<16>(p, block - shared_items, G, it)) {
        const uint32_t ring = smem_addr(smem);
        if (tid == 0) {
            for (int i = 0; i < kStages; ++i) {
                mbar_init(smem_addr(&sync.full[i]), 1);
                mbar_init(smem_addr(&sync.empty[i]), kWarps);
            }
            sync.gave_up = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
        bool ok;
        if (warp == kWarps) {
            ok = fill<D, kStages>(&map_k, &map_v, p, it, kvh, page_shift, bounds, ring, sync);
        } else {
            ok = family ? attend<D, ROW_TILES, kStages>(q, partial, p, it, kvh, G, ring, smem, sync)
                        : attend<D, 1, kStages>(q, partial, p, it, kvh, G, ring, smem, sync);
        }
        if (!ok && (tid & 31) == 0) { *(volatile int*)&sync.gave_up = 1; atomicMax(error, warp == kWarps ? 2u : 4u); }
        __syncthreads();
        if (*(volatile int*)&sync.gave_up) {
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);                     // copies in flight land before this block's memory is reused
        }
    }
    // complete no sooner than the kernel it ran beside: the last block alone waits, the others leave their places to those behind them
    if (beside && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// Joins a row's parts: a warp per row, a lane per part for their weights and per four dimensions for the sums.  A sequence outside
// the families has no shared parts.  Latency bounds it: 7 us for 3,232 rows whose parts are cold.
template <typename T>
__global__ void __launch_bounds__(kThreads)
shared_join_kernel(const float* __restrict__ partial, T* __restrict__ out, const Shared p, int rows, int D, int shared_tile) {
    const int row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    const int room = p.n_shared + p.n_own, stride = D + 2, seq = row / p.Hq;
    // (lengths were there before the kernels ahead began)
    int shared = 0;
    if (p.n_families > 0) {
        const int keys = shared_keys(p, seq), chunk = shared_chunk(p, keys, shared_tile);
        shared = (keys + chunk - 1) / chunk;
    }
    const int parts = shared + own_parts(p, seq), skipped = p.n_shared - shared;  // part i stands at i, or, of its own, at i + skipped
    const float* base = partial + (size_t)row * room * stride;
    pdl_wait();
    float m[2], l[2];                                                             // up to 64 parts
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        const float2 ml = i < parts ? *reinterpret_cast<const float2*>(base + (size_t)(i < shared ? i : i + skipped) * stride + D) : make_float2(-INFINITY, 0.0f);
        m[h] = ml.x;
        l[h] = ml.y;
    }
    float top = warp_max(fmaxf(m[0], m[1]));
    if (top == -INFINITY) top = 0.0f;                    // nothing to attend to (or NaN, which l carries)
    m[0] = pow2(m[0] - top);
    m[1] = pow2(m[1] - top);
    const float sum = warp_sum(l[0] * m[0] + l[1] * m[1]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // a sequence without keys: zeros
    for (int d0 = 0; d0 < D; d0 += 128) {
        const int d = d0 + lane * 4;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < parts; i0 += 8) {          // eight parts on their way at once (those beyond the last weigh nothing)
            float2 a[8], b[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u;
                const float* part = base + (size_t)(i < shared ? i : i + skipped) * stride + d;
                a[u] = b[u] = make_float2(0.0f, 0.0f);
                if (i < parts && d < D) {
                    a[u] = *reinterpret_cast<const float2*>(part);
                    b[u] = *reinterpret_cast<const float2*>(part + 2);
                }
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u;
                const float f = __shfl_sync(0xffffffffu, i < 32 ? m[0] : m[1], i & 31);
                acc[0] = fmaf(a[u].x, f, acc[0]); acc[1] = fmaf(a[u].y, f, acc[1]); acc[2] = fmaf(b[u].x, f, acc[2]); acc[3] = fmaf(b[u].y, f, acc[3]);
            }
        }
        if (d < D) {
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] *= inv;
            store_quad(out + (size_t)row * D + d, acc);
        }
    }
}

template <typename T, int QUADS>
int launch_general(const void* q, const void* k_pool, const void* v_pool, float* partial, const Shared& p, int D, int G, cudaStream_t stream) {
    const long long shared = family_blocks(p, G, kRows), all = (shared + own_blocks(p, G, kRows)) * p.Hkv;
    if (all > 0x7fffffff) return PB_ERR_TOO_LARGE;
    const size_t smem = general_smem<T>(D);
    static SmemLimit limit;
    if (const int rc = limit.allow(shared_general_kernel<T, QUADS>, smem)) return rc;
    shared_general_kernel<T, QUADS><<<(unsigned)all, kThreads, smem, stream>>>((const T*)q, (const T*)k_pool, (const T*)v_pool, partial, p,
                                                                                           (int)shared, D, pool_bounds_now());
    return launch_status();
}

// A pool as rows of D dimensions, a box a page of 64 of them.
int make_map(CUtensorMap* map, const void* pool, long long rows, int D, int page_size) {
    EncodeTiledFn encode = encode_fn();
    if (!encode) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)page_size};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pool), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : PB_ERR_BAD_SIZE;
}

template <int D, int ROW_TILES>
int launch_tc(const void* q, const Maps& maps, float* partial, const Shared& p, int G, bool beside, cudaStream_t stream) {
    const long long shared = family_blocks(p, G, ROW_TILES * 16), items = (shared + own_blocks(p, G, 16)) * p.Hkv;
    if (items > 0x7fffffff) return PB_ERR_TOO_LARGE;
    constexpr int smem = kRing<ROW_TILES> + 1024;
    static_assert(kWarps * 16 * (D + 8) * 4 <= kRing<ROW_TILES>, "the warps meet in the ring's memory");
    static SmemLimit limit;
    static DeviceLimit most;
    if (const int rc = limit.allow(shared_tc_kernel<D, ROW_TILES>, smem)) return rc;
    if (const int rc = share_most(most, shared_tc_kernel<D, ROW_TILES>)) return rc;
    return launch_early(beside, shared_tc_kernel<D, ROW_TILES>, dim3((unsigned)items), dim3(kTcThreads), smem, stream, (const bf16*)q,
                        maps.k, maps.v, partial, p, (int)shared, log2_exact(p.page_size), pool_bounds_now(), maps.error, beside);
}

// Families of up to 16 rows meet their keys as a sequence its own.  Beyond that heads of 128 take the tcgen05 kernel for the shared sides
// (one family over 4,000 keys, 4 heads a member, us in all: 8 members 13 against 20, 64 members 26 against 49), which takes no other; heads of 64 as many row tiles as the
// largest family fills.  The tcgen05 kernel finds maxima and masks keys before it scales, which is right for a scale above 0 alone: the others
// take the rest.
bool tcgen05_takes(int rows, int D, float scale_log2) { return D == 128 && rows > 16 && scale_log2 > 0.0f; }

int launch_tc(const void* q, const void* k_pool, const void* v_pool, float* partial, Shared p, int G, int D, int n_pages, unsigned int* error,
              cudaStream_t stream) {
    Maps maps;
    maps.error = error;
    const long long pool_rows = (long long)n_pages * p.Hkv * p.page_size;
    if (pool_rows > 0x7fffffff) return PB_ERR_TOO_LARGE;
    int rc = make_map(&maps.k, k_pool, pool_rows, D, p.page_size);
    if (rc == 0) rc = make_map(&maps.v, v_pool, pool_rows, D, p.page_size);
    if (rc != 0) return rc;
    const int rows = p.n_families > 0 ? p.most_members * G : 0;
    if (tcgen05_takes(rows, D, p.scale_log2)) {
        rc = launch_tcgen05(q, maps, partial, p, stream);
        if (rc != 0) return rc;
        p.n_families = 0;                                 // (n_shared stays: it is where a sequence's own parts begin)
        return launch_tc<128, 1>(q, maps, partial, p, G, true, stream);
    }
    if (D == 128) return launch_tc<128, 1>(q, maps, partial, p, G, false, stream);
    if (rows <= 16) return launch_tc<64, 1>(q, maps, partial, p, G, false, stream);
    if (rows <= 32) return launch_tc<64, 2>(q, maps, partial, p, G, false, stream);
    return launch_tc<64, 4>(q, maps, partial, p, G, false, stream);
}

bool tc_takes(int dtype, int D, int page_size) {
    return dtype == PB_BF16 && (D == 64 || D == 128) && log2_exact(page_size) >= 3 && page_size <= kTile;
}

}  // namespace

// Query rows that a block of the shared sides works on (for a scale above 0): what the caller cuts the keys by.
PB_EXPORT int pb_shared_rows(int dtype, int rows, int D, int page_size) {
    if (!tc_takes(dtype, D, page_size)) return kRows;
    return tcgen05_takes(rows, D, 1.0f) ? kTcgen05Rows : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

// q, out [n_seqs, Hq, D], pools [pages, Hkv, page_size, D] (dtype 0 float32, 1 bfloat16); block_table int32 [n_seqs, table_stride];
// kv_len, shared_len int32 [n_seqs]; members int32 [n_members], family_start int32 [n_families + 1]; partial float32
// [n_seqs * Hq * (n_shared + n_own) * (D + 2)], all 16-byte aligned; n_pages: of the pools; error: the word that a block sets which gave up
// a bounded wait; own_chunk: keys of a part of a sequence's own, a multiple of 64 and of the page; n_shared + n_own <= 64.
PB_EXPORT int pb_paged_attention_shared(int dtype, const void* q, const void* k_pool, const void* v_pool, void* out, float* partial,
                                        const int* block_table, int table_stride, const int* kv_len, const int* shared_len, const int* members,
                                        const int* family_start, int n_seqs, int n_members, int n_families, int most_members, int Hq, int Hkv, int D,
                                        int page_size, float scale, int n_shared, int n_own, int own_chunk, int n_pages, unsigned int* error,
                                        cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (dtype != PB_F32 && dtype != PB_BF16) return PB_ERR_BAD_DTYPE;
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || D % 16 || D > 256 || page_size <= 0 || table_stride <= 0) return PB_ERR_BAD_SIZE;
    if (n_families < 0 || most_members < 0 || n_members < 0 || n_own <= 0 || n_shared < 0 || (n_families > 0 && n_shared == 0)) return PB_ERR_BAD_SIZE;
    if (own_chunk <= 0 || own_chunk % 64 || own_chunk % page_size) return PB_ERR_BAD_SIZE;
    if (Hkv > 65535 || n_shared + n_own > 64 || (long long)n_seqs * Hq > 0x7fffffff) return PB_ERR_TOO_LARGE;
    const int G = Hq / Hkv;
    Shared p{block_table, kv_len, shared_len, members, family_start, n_seqs, n_members, n_families, most_members, table_stride, Hq, Hkv, page_size, n_shared, n_own,
             own_chunk, scale * kLog2e};
    int rc;
    if ((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out | (uintptr_t)partial) & 15) != 0) return PB_ERR_BAD_SIZE;
    if (tc_takes(dtype, D, page_size) && n_pages > 0 && error != nullptr)
        rc = launch_tc(q, k_pool, v_pool, partial, p, G, D, n_pages, error, stream);
    else if (dtype == PB_F32)
        rc = D <= 128 ? launch_general<float, 1>(q, k_pool, v_pool, partial, p, D, G, stream) : launch_general<float, 2>(q, k_pool, v_pool, partial, p, D, G, stream);
    else
        rc = D <= 128 ? launch_general<bf16, 1>(q, k_pool, v_pool, partial, p, D, G, stream) : launch_general<bf16, 2>(q, k_pool, v_pool, partial, p, D, G, stream);
    if (rc != 0) return rc;
    const int rows = n_seqs * Hq, blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
    static_assert(kKeys == kTile, "the parts of a family's keys are cut by the same tile in both");
    const int shared_tile = tc_takes(dtype, D, page_size) && tcgen05_takes(most_members * G, D, p.scale_log2) ? kTcgen05Rows : kTile;
    if (dtype == PB_F32) return launch_pdl(shared_join_kernel<float>, dim3(blocks), dim3(kThreads), 0, stream, partial, (float*)out, p, rows, D, shared_tile);
    return launch_pdl(shared_join_kernel<bf16>, dim3(blocks), dim3(kThreads), 0, stream, partial, (bf16*)out, p, rows, D, shared_tile);
}

// A new limit of this kernel's bounded waits in clock cycles.
PB_EXPORT int pb_shared_wait_limit(long long limit) {
    return limit > 0 && cudaMemcpyToSymbol(g_wait_limit, &limit, sizeof(limit)) == cudaSuccess ? 0 : -1;
}

// Lets one of these waits run out: afterwards the error word reads 9.  Set a short limit first.
namespace {
struct SharedUnit {};
}
PB_EXPORT int pb_shared_wait_selftest(unsigned int* error, cudaStream_t stream) {
    if (error == nullptr) return PB_ERR_BAD_SIZE;
    wait_gives_up_kernel<SharedUnit><<<1, 32, 0, stream>>>(error);
    return launch_status();
}
