// Log probability of given tokens and entropy straight from hidden rows h [R, K] and the head's weight W [V, K] in bfloat16: the logits
// x = cap tanh(scale (h W^T) / cap) exist only in tensor memory.
//
// The product is tcgen05.mma with rows of h as the lanes of the accumulator and vocabulary entries as its columns, so a row's sums (see
// scores.cuh) are one thread's own: an epilogue thread walks over its row's columns of a tile and keeps maximum, sum and weighted sum,
// without a word to its neighbours.  A tile leaves three numbers per row; a second kernel joins a row's tiles.
//
// Bound: with few rows the bytes of W, with many the products (2 R V K).  The epilogue of a tile costs some 3,000 cycles beside the
// 32,768 that the products of 128 rows, 256 columns and K = 4096 take on one SM, and runs under those of the next tile: there are two
// accumulators.  Roles, ring of stages and bounded waits are those of gemm_tcgen05.cu.
//
// Up to 128 rows a block per SM streams W (once, so it is the first to leave L2: 201 against 206 us for 17 rows of 4,096 against 151,936,
// 206 against 216 for 100).  More rows go to pairs of blocks on tiles of 256 rows (cta_group::2): each block brings its own 128 rows of h and
// half of the tile's columns of W, which so crosses from L2 once a pair (2,048 rows: 1,885 us, single blocks 1,949).
//
// Measured with K = 4096 and V = 151,936: 17 rows 200 us (6.2 TB/s), 2,048 rows 1,850 us (1,380 TFLOP/s; the tensor pipe is active 87 % of
// the time).  The products' sums are kept in the tensor cores' float32, which cut off where others round: a log probability is some 7e-7 of
// itself away from sums in 64 bits.
//
// The width of a tile is chosen so that the tiles fill the SMs in whole rounds (see plan()).
#include "scores.cuh"
#include "tcgen05_common.cuh"

namespace {

using namespace pb;
typedef __nv_bfloat16 bf16;

constexpr int kBM = 128;                     // rows of h per tile: lanes of tensor memory
constexpr int kMostColumns = 256;            // of a tile: columns of one of the two accumulators
constexpr int kBK = 64;                      // k per stage: one 128-byte swizzle atom
constexpr int kThreads = 192;                // producer warp, MMA warp, four epilogue warps
constexpr int kTmemColumns = 512;
constexpr int kMostStages = 8;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kSmem = 226 * 1024;
constexpr uint32_t kPeerBitMask = 0xFEFFFFFFu;   // clears the bit in which the two blocks' shared-memory addresses differ: rank 0's barrier

struct HeadArgs {
    const int* tokens;          // [rows]
    float* part;                // [3][n_tiles][rows]: m, s, t
    float* given;               // [rows]: the given token's logit
    unsigned int* error;        // set when a bounded wait ran out
    int rows, vocab, k;
    int columns;                // of a tile
    int m_tiles, n_tiles, stages;
    int stage_bytes;
    float scale, cap;           // cap 0: none
};

__device__ __forceinline__ uint64_t umma_desc(uint32_t addr) {      // K-major, 128-byte rows, 128-byte swizzle
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3fff);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <bool PAIR>
__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on `bar` (of both blocks of a pair) once the products issued so far have retired.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((unsigned short)3) : "memory");
    else
        umma_commit(bar);
}
// A box into this block's shared memory; its bytes count on `bar`, in a pair on rank 0's.
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar & kPeerBitMask), "r"(c0), "r"(c1) : "memory");
    else
        tma_load_2d(dst, map, bar, c0, c1);
}
// The same for bytes that are read once and should be the first to leave L2.
__device__ __forceinline__ void load_box_once(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "l"(policy) : "memory");
}
__device__ __forceinline__ void both_blocks() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One row's columns [first, first + columns) of an accumulator.
template <bool CAP>
__device__ __forceinline__ void score_tile(const HeadArgs& p, uint32_t taddr, int first, int token, Stats& st, float& given) {
#pragma unroll 1
    for (int c = 0; c < p.columns; c += 32) {
        uint32_t v[32];
        tmem_ld32(taddr + c, v);
        float x[32];
        const int n0 = first + c, valid = min(p.columns - c, p.vocab - n0);         // (a tile may end inside the 32 columns)
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            x[i] = __uint_as_float(v[i]) * p.scale;
            if (CAP) x[i] = p.cap * tanhf(x[i] / p.cap);
        }
        if (valid < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i >= valid) x[i] = -INFINITY;
        }
        add_logits(st, x);
        if (__any_sync(0xffffffffu, token >= n0 && token < n0 + valid)) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (token == n0 + i && i < valid) given = x[i];
        }
    }
}

// PAIR: a cluster of two blocks per tile of 256 rows; barriers as in gemm_tcgen05.cu: "full" and "accumulator empty" are rank 0's, which
// issues the products of both.
template <bool CAP, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
head_scores_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, const HeadArgs p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[2 * kMostStages + 4];                 // full, empty, accumulator full, accumulator empty
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;

    pdl_trigger();                                                               // (what joins the tiles waits for this kernel's end)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t rank = 0;
    if (PAIR) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
    constexpr int kRows = PAIR ? 2 * kBM : kBM;                                  // of a tile
    const int own_columns = PAIR ? p.columns / 2 : p.columns;                    // of W that this block brings
    const int k_tiles = (p.k + kBK - 1) / kBK;
    const int total_tiles = p.m_tiles * p.n_tiles;
    const uint32_t full0 = smem_addr(bars), empty0 = smem_addr(bars + kMostStages);
    const uint32_t acc_full0 = smem_addr(bars + 2 * kMostStages), acc_empty0 = smem_addr(bars + 2 * kMostStages + 2);

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(acc_full0 + 8 * a, 1); mbar_init(acc_empty0 + 8 * a, PAIR ? 8 : 4); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) both_blocks();                                                     // the peer's barriers exist before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            uint64_t once = 0;
            if (!PAIR) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
            int s = 0, turn = 0;
            bool ok = true;
            for (int tile = worker; tile < total_tiles && ok; tile += workers) {
                const int m0 = (tile % p.m_tiles) * kRows + (int)rank * kBM, n0 = (tile / p.m_tiles) * p.columns + (int)rank * own_columns;
                for (int kt = 0; kt < k_tiles; ++kt) {
                    if (!mbar_wait(empty0 + 8 * s, (turn & 1) ^ 1, abort_flag)) { ok = false; break; }
                    const uint32_t dst = smem_addr(smem) + s * p.stage_bytes;
                    const uint32_t bytes = (uint32_t)p.stage_bytes;
                    if (rank == 0) mbar_expect_tx(full0 + 8 * s, PAIR ? 2 * bytes : bytes);
                    load_box<PAIR>(dst, &map_h, full0 + 8 * s, kt * kBK, m0);
                    if (PAIR) load_box<PAIR>(dst + kABytes, &map_w, full0 + 8 * s, kt * kBK, n0);
                    else load_box_once(dst + kABytes, &map_w, full0 + 8 * s, kt * kBK, n0, once);
                    if (++s == p.stages) { s = 0; ++turn; }
                }
            }
            if (!ok) { *abort_flag = 1; atomicMax(p.error, 2u); }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
            const uint64_t desc0 = umma_desc(smem_addr(smem));
            // float32 accumulator, bfloat16 operands, both K-major, columns >> 3, rows >> 4
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.columns >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
            int s = 0, turn = 0, j = 0;
            bool ok = true;
            for (int tile = worker; tile < total_tiles && ok; tile += workers, ++j) {
                const int acc = j & 1;
                ok = mbar_wait(acc_empty0 + 8 * acc, ((j >> 1) & 1) ^ 1, abort_flag);
                const uint32_t tmem_d = tmem_u + acc * kMostColumns;
                for (int kt = 0; kt < k_tiles && ok; ++kt) {
                    if (!mbar_wait(full0 + 8 * s, turn & 1, abort_flag)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t a_desc = desc0 + (uint64_t)((uint32_t)s * (uint32_t)(p.stage_bytes >> 4));
                    const uint64_t b_desc = a_desc + (uint64_t)(kABytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)
                            umma_bf16<PAIR>(tmem_d, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc, (kt > 0 || k > 0) ? 1u : 0u);
                        commit<PAIR>(empty0 + 8 * s);
                        if (kt == k_tiles - 1) commit<PAIR>(acc_full0 + 8 * acc);
                    }
                    __syncwarp();
                    if (++s == p.stages) { s = 0; ++turn; }
                }
            }
            if (!ok && lane == 0) { *abort_flag = 1; atomicMax(p.error, 3u); }
        }
    } else {
        const int quarter = warp & 3;
        int j = 0;
        for (int tile = worker; tile < total_tiles; tile += workers, ++j) {
            const int acc = j & 1;
            const int m0 = (tile % p.m_tiles) * kRows + (int)rank * kBM, nt = tile / p.m_tiles;
            if (!mbar_wait(acc_full0 + 8 * acc, (j >> 1) & 1, abort_flag)) {
                if (lane == 0) { *abort_flag = 1; atomicMax(p.error, 4u); }
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int row = m0 + quarter * 32 + lane;
            if (m0 + quarter * 32 < p.rows) {                         // a warp without rows has nothing to read
                const int token = row < p.rows ? p.tokens[row] : -1;
                Stats st = {-INFINITY, 0.0f, 0.0f};
                float given = 0.0f;
                const int first = nt * p.columns;
                score_tile<CAP>(p, tmem_base + acc * kMostColumns + ((uint32_t)(quarter * 32) << 16), first, token, st, given);
                if (row < p.rows) {
                    const size_t plane = (size_t)p.n_tiles * p.rows, at = (size_t)nt * p.rows + row;
                    p.part[at] = st.m;
                    p.part[at + plane] = st.s;
                    p.part[at + 2 * plane] = st.t;
                    if (token >= first && token < min(first + p.columns, p.vocab)) p.given[row] = given;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (PAIR)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"((acc_empty0 + 8 * acc) & kPeerBitMask) : "memory");
                else
                    mbar_arrive(acc_empty0 + 8 * acc);
            }
        }
    }
    __syncwarp();
    if (*abort_flag) {
        // a role gave up: give copies and products that are still in flight time to land before this block's memory is reused
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) both_blocks();                                                     // neither leaves while the other may still touch its memory
    if (warp == 1) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns));
    }
}

// Joins the tiles of eight rows per block: 64 threads a row take turns at its tiles.
constexpr int kJoinRows = 8, kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads)
head_join_kernel(const float* __restrict__ part, const float* __restrict__ given, const int* __restrict__ tokens, float* __restrict__ logprob,
                 float* __restrict__ entropy, int rows, int n_tiles, int vocab) {
    __shared__ Stats st_s[kJoinThreads / 32][kJoinRows];
    const int tid = threadIdx.x, warp = tid >> 5, i = tid % kJoinRows, row = blockIdx.x * kJoinRows + i;
    const size_t plane = (size_t)n_tiles * rows;
    pdl_wait();
    Stats st = {-INFINITY, 0.0f, 0.0f};
    if (row < rows) {
#pragma unroll 4
        for (int tile = tid / kJoinRows; tile < n_tiles; tile += kJoinThreads / kJoinRows) {
            const float* at = part + (size_t)tile * rows + row;
            st = join(st, Stats{at[0], at[plane], at[2 * plane]});
        }
    }
#pragma unroll
    for (int o = kJoinRows; o < 32; o <<= 1)
        st = join(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.t, o)});
    if ((tid & 31) < kJoinRows) st_s[warp][i] = st;
    __syncthreads();
    if (tid >= kJoinRows || row >= rows) return;
    for (int w = 1; w < kJoinThreads / 32; ++w) st = join(st, st_s[w][i]);
    const int token = tokens[row];
    const float log_s = logf(st.s);
    logprob[row] = token >= 0 && token < vocab ? (given[row] - st.m) - log_s : nanf("");
    entropy[row] = log_s - st.t / st.s;
}

int sm_count() {
    static int n = [] {
        int dev = 0, v = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 0;
        return v > 0 ? v : 148;
    }();
    return n;
}

struct Plan {
    bool pair;
    int columns, m_tiles, n_tiles;
};

// The widest tile whose rounds over the SMs (pairs of them) come out even: all tiles are as wide, so the time is rounds x (columns + what a
// tile costs besides, about 16 columns' worth).  (17 rows against 151,936: 731 tiles of 208 in five rounds, 201 us;
// 594 of 256 take five as well, 220.)
Plan plan(int rows, int vocab) {
    Plan best = {};
    best.pair = rows > kBM;
    const int tile_rows = best.pair ? 2 * kBM : kBM, step = best.pair ? 32 : 16, workers = best.pair ? sm_count() / 2 : sm_count();
    best.m_tiles = (rows + tile_rows - 1) / tile_rows;
    long long least = 0;
    for (int columns = kMostColumns; columns >= step; columns -= step) {
        const long long tiles = (long long)best.m_tiles * ((vocab + columns - 1) / columns);
        const long long cost = (tiles + workers - 1) / workers * (columns + 16);
        if (least == 0 || cost < least) {
            least = cost;
            best.columns = columns;
        }
    }
    best.n_tiles = (vocab + best.columns - 1) / best.columns;
    return best;
}

// Row-major [rows, k] bfloat16 matrix, boxes of box_rows x 64, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, const void* base, int rows, int k, int box_rows) {
    EncodeTiledFn encode = encode_fn();
    if (!encode) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)k * 2};
    const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : PB_ERR_BAD_SIZE;
}

template <bool CAP, bool PAIR>
int launch(const CUtensorMap& mh, const CUtensorMap& mw, const HeadArgs& p, cudaStream_t stream) {
    static SmemLimit limit;
    if (const int rc = limit.allow(head_scores_kernel<CAP, PAIR>, kSmem)) return rc;
    const long long tiles = (long long)p.m_tiles * p.n_tiles, workers = PAIR ? sm_count() / 2 : sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles < workers ? tiles : workers) * (PAIR ? 2 : 1));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.stages * p.stage_bytes + 1024;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, head_scores_kernel<CAP, PAIR>, mh, mw, p);
}

}  // namespace

// 1 if pb_head_scores takes these sizes (rows of K elements are whole multiples of 16 bytes, as TMA's strides have to be).
PB_EXPORT int pb_head_scores_supported(int rows, int vocab, int k) {
    return rows > 0 && vocab > 0 && k > 0 && k % 8 == 0 && (long long)rows * vocab / 16 < 0x7fffffff ? 1 : 0;
}

// float32 elements of scratch that pb_head_scores needs.
PB_EXPORT long pb_head_scores_scratch(int rows, int vocab) { return (long)(3LL * plan(rows, vocab).n_tiles + 1) * rows; }

// A new limit of this kernel's bounded waits in clock cycles.
PB_EXPORT int pb_head_scores_wait_limit(long long limit) {
    return limit > 0 && cudaMemcpyToSymbol(g_wait_limit, &limit, sizeof(limit)) == cudaSuccess ? 0 : -1;
}

// Lets one of these waits run out: afterwards the error word reads 9.  Set a short limit first.
namespace {
struct HeadScoresUnit {};
}
PB_EXPORT int pb_head_scores_wait_selftest(unsigned int* error, cudaStream_t stream) {
    if (error == nullptr) return PB_ERR_BAD_SIZE;
    wait_gives_up_kernel<HeadScoresUnit><<<1, 32, 0, stream>>>(error);
    return launch_status();
}

// h [rows, k], w [vocab, k] bfloat16, 16-byte aligned; tokens int32 [rows]; logprob, entropy float32 [rows]; scratch float32 of
// pb_head_scores_scratch elements; error: the word that a block sets which gave up a bounded wait.  cap 0: none.
PB_EXPORT int pb_head_scores(const void* h, const void* w, const int* tokens, float* logprob, float* entropy, int rows, int vocab, int k, float scale,
                             float cap, float* scratch, unsigned int* error, cudaStream_t stream) {
    if (!pb_head_scores_supported(rows, vocab, k) || (((uintptr_t)h | (uintptr_t)w) & 15) != 0 || error == nullptr || !(cap >= 0.0f)) return PB_ERR_BAD_SIZE;
    const Plan at = plan(rows, vocab);
    const int own_columns = at.pair ? at.columns / 2 : at.columns;
    HeadArgs p = {tokens, scratch, scratch + 3 * (size_t)at.n_tiles * rows, error, rows, vocab, k, at.columns, at.m_tiles, at.n_tiles, 0,
                  kABytes + own_columns * kBK * 2, scale, cap};
    const int stages = (kSmem - 1024) / p.stage_bytes;
    p.stages = stages < kMostStages ? stages : kMostStages;
    CUtensorMap mh, mw;
    int rc = make_map(&mh, h, rows, k, kBM);
    if (rc == 0) rc = make_map(&mw, w, vocab, k, own_columns);
    if (rc == 0 && at.pair) rc = cap > 0.0f ? launch<true, true>(mh, mw, p, stream) : launch<false, true>(mh, mw, p, stream);
    else if (rc == 0) rc = cap > 0.0f ? launch<true, false>(mh, mw, p, stream) : launch<false, false>(mh, mw, p, stream);
    if (rc != 0) return rc;
    return launch_pdl(head_join_kernel, dim3((rows + kJoinRows - 1) / kJoinRows), dim3(kJoinThreads), 0, stream, (const float*)p.part, (const float*)p.given, tokens,
                      logprob, entropy, rows, at.n_tiles, vocab);
}
