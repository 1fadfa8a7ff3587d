// The shared sides of the attention over a forked cache (attention_shared.cu) on the fifth-generation tensor cores: bfloat16, head size 128,
// pages of 8, 16, 32 or 64 keys.
//
// A block has up to 128 query rows of a family (members x the group's heads) and one split of the family's shared keys.  The rows are the
// lanes of tensor memory: S = Q K^T (tcgen05.mma, 128 x 128 x 16 steps, operands in shared memory), a thread per row takes its row of S,
// keeps maximum and sum in float32 and writes P = 2^(s c - m c), rounded to bfloat16 as the product's operand has to be (2^-9 of each weight, the sum is
// of the unrounded ones), over S; O += P V reads P from tensor memory and V as it
// lies in the pages.  The product costs the same for one row as for 128, so a key tile passes the tensor cores once however many of the
// family's sequences there are: bound by the bytes of the keys and values.  (mma.sync takes 2,100 cycles for 32 rows x 64 keys, with two
// blocks an SM as long as the bytes do, and so many times that for larger families.)
//
// A thread takes 128 exponentials a tile, 1,900 cycles with all that goes with them, more than the tile's bytes take where SMs are idle.  So
// families of up to 64 rows stand in tensor memory twice, of up to 32 four times: each copy has its own half or quarter of a tile's keys,
// writes zeros for the weights of the others, and the copies' sums are joined at the end (REPEAT; zero times an infinite value is NaN).  (12 families of 8, 32 rows per kv head,
// over up to 2,600 keys, 92 MB: 31 us cold.)
//
// Roles: warps 0-3 softmax (and the gathering of the query rows, which lie with their sequences), warp 4 issues the products, warp 5 brings K
// and warp 6 V, a lane per half page.  S has two buffers, S of the next tile is issued before O += P V of this one.  The maximum moves only
// when it grew by more than 2^8; O is rescaled in tensor memory only then, and the sums use the same maximum.  Maxima and masks are those of
// unscaled scores: the scale is above 0 (launch_tc sees to it).
//
// Shared keys are whole pages, so a page that is read holds nothing but keys.  Where the last tile has fewer pages, the columns of S are
// masked, and V's buffer is zero or holds an earlier tile's values there.
//
// Every wait is bounded by a clock limit; a role that gives up sets the error word, the block lets its copies land, frees its tensor memory
// and returns.
#include "attention_shared.cuh"
#include "attention_tcgen05.cuh"

namespace {

using namespace pb;
using namespace pb::attn5;
using namespace pb::shared_attention;

constexpr int kThreads = 224;
// K tiles, and V tiles, on their way: what is left of an SM takes a block of the own sides' kernel.  (Three: 47.6 against 48.4 us for 101 sequences with
// own keys of up to 500, 45.3 against 45.0 for 32 of up to 2,000.)
constexpr int kStages = 2;
constexpr int kSmemBytes = (1 + 2 * kStages) * kTileBytes + 1024;
constexpr int kTmemColumns = 512;                // S[0] | S[1] | O, and what is left of a power of two

struct Sync {
    uint64_t q_full, o_full, o_done, s_full[2], p_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint32_t tmem;
    int gave_up;
};

// The four softmax warps meet here.
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int REPEAT>
__global__ void __launch_bounds__(kThreads, 1)
shared_tcgen05_kernel(const bf16* __restrict__ q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      float* __restrict__ partial, const Shared p, int page_shift, const PoolBounds bounds, unsigned int* error) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = smem;
    unsigned char* k_s = smem + kTileBytes;
    unsigned char* v_s = k_s + kStages * kTileBytes;
    __shared__ Sync sync;
    pdl_trigger();                               // launched the ordinary way: the sequences' own sides may run beside it
    const int G = p.Hq / p.Hkv, kvh = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* abort_flag = &sync.gave_up;
    Item it;
    if (!family_item<kBM / REPEAT, kBN>(p, blockIdx.x, G, it)) return;
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sync.tmem)), "r"(kTmemColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    const int n_tiles = (it.end - it.begin + kBN - 1) / kBN;              // (a split begins at a multiple of kBN)
    // softmax warp w has rows (w % kGroups) * 32 .. and copy w / kGroups of them
    constexpr int kGroups = 4 / REPEAT, kKeys = kBN / REPEAT;
    const int active = (it.rows + 31) / 32 * REPEAT;                      // softmax warps that have rows
    if (tid == 128) {
        mbar_init(smem_addr(&sync.q_full), 4);
        mbar_init(smem_addr(&sync.o_full), 1);
        mbar_init(smem_addr(&sync.o_done), 1);
        for (int i = 0; i < 2; ++i) { mbar_init(smem_addr(&sync.s_full[i]), 1); mbar_init(smem_addr(&sync.p_full[i]), max(1, active)); }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_addr(&sync.k_full[i]), 1); mbar_init(smem_addr(&sync.k_empty[i]), 1);
            mbar_init(smem_addr(&sync.v_full[i]), 1); mbar_init(smem_addr(&sync.v_empty[i]), 1);
        }
        sync.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // values of the last tile that no page brings, where no earlier tile has been
    const int last_rows = it.end - it.begin - (n_tiles - 1) * kBN;
    if (n_tiles > 0 && n_tiles <= kStages && last_rows < kBN) {
        unsigned char* tile = v_s + (n_tiles - 1) * kTileBytes;
        for (int i = tid; i < (kBN - last_rows) * 16; i += kThreads)
            *reinterpret_cast<uint4*>(tile + (i & 8 ? kHalfBytes : 0) + (last_rows + (i >> 4)) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem_s = sync.tmem, tmem_o = tmem_s + 2 * kBN;

    if (warp >= 5) {
        // ---------------- TMA: a lane per half page of a tile
        const bool for_v = warp == 6;
        unsigned char* tiles = for_v ? v_s : k_s;
        const CUtensorMap* map = for_v ? &map_v : &map_k;
        uint64_t* full = for_v ? sync.v_full : sync.k_full;
        uint64_t* empty = for_v ? sync.v_empty : sync.k_empty;
        const int slot = lane >> 1, half = lane & 1, page_size = 1 << page_shift;
        bool ok = true;
        for (int j = 0; j < n_tiles && ok; ++j) {
            const int st = j % kStages, key = it.begin + j * kBN + (slot << page_shift);
            const bool want = slot < (kBN >> page_shift) && key < it.end;
            int page = want ? it.table[key >> page_shift] : 0;
            if (!page_ok(page, bounds)) page = 0;
            const uint32_t n_want = __popc(__ballot_sync(0xffffffffu, want));
            if (lane == 0) {
                ok = mbar_wait(smem_addr(&empty[st]), ((j / kStages) & 1) ^ 1, abort_flag);
                if (ok) mbar_expect_tx(smem_addr(&full[st]), n_want * (uint32_t)page_size * 128u);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (ok && want)
                tma_load_2d(smem_addr(tiles) + st * kTileBytes + half * kHalfBytes + (slot << page_shift) * 128, map, smem_addr(&full[st]), half * 64,
                            (page * p.Hkv + kvh) << page_shift);
            __syncwarp();
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicMax(error, 2u); }
    } else if (warp == 4) {
        // ---------------- MMA issuer: the warp walks the loop uniformly, one elected lane issues
        const uint32_t ts = __shfl_sync(0xffffffffu, tmem_s, 0), to = ts + 2 * kBN;
        const uint64_t q_desc = desc_k_major(smem_addr(q_s)), k_desc = desc_k_major(smem_addr(k_s)), v_desc = desc_mn_major(smem_addr(v_s));
        auto issue_s = [&](int j) -> bool {
            const int st = j % kStages;
            if (!mbar_wait(smem_addr(&sync.k_full[st]), (j / kStages) & 1, abort_flag)) return false;
            fence_after();
            const uint64_t kd = k_desc + (uint64_t)((uint32_t)st * (kTileBytes >> 4));
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < kD / 16; ++ks) {
                    const uint32_t off = (uint32_t)(ks >> 2) * (kHalfBytes >> 4) + (uint32_t)(ks & 3) * 2u;
                    umma_ss(ts + (uint32_t)(j & 1) * kBN, q_desc + off, kd + off, kIdescS, ks > 0 ? 1u : 0u);
                }
                umma_commit(smem_addr(&sync.k_empty[st]));
                umma_commit(smem_addr(&sync.s_full[j & 1]));
            }
            __syncwarp();
            return true;
        };
        bool ok = n_tiles == 0 || (mbar_wait(smem_addr(&sync.q_full), 0, abort_flag) && issue_s(0));
        for (int j = 0; j < n_tiles && ok; ++j) {
            if (j + 1 < n_tiles && !issue_s(j + 1)) { ok = false; break; }
            const int st = j % kStages;
            if (!mbar_wait(smem_addr(&sync.v_full[st]), (j / kStages) & 1, abort_flag) || !mbar_wait(smem_addr(&sync.p_full[j & 1]), (j >> 1) & 1, abort_flag)) {
                ok = false;
                break;
            }
            fence_after();
            const uint64_t vd = v_desc + (uint64_t)((uint32_t)st * (kTileBytes >> 4));
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kBN / 16; ++kk)
                    umma_ts(to, ts + (uint32_t)(j & 1) * kBN + (uint32_t)kk * 8u, vd + (uint64_t)(kk * (2048 >> 4)), kIdescPV, (j > 0 || kk > 0) ? 1u : 0u);
                umma_commit(smem_addr(&sync.v_empty[st]));
                umma_commit(smem_addr(&sync.o_full));
                if (j + 1 == n_tiles) umma_commit(smem_addr(&sync.o_done));
            }
            __syncwarp();
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicMax(error, 3u); }
    } else {
        // ---------------- softmax: thread r owns lane r of tensor memory, a copy of a query row
        const int r = warp * 32 + lane, i = warp % kGroups * 32 + lane, copy = warp / kGroups;
        const bool has_rows = warp % kGroups * 32 < it.rows;
        int row = -1;                                             // sequence * Hq + head
        if (i < it.rows) {
            const int seq = it.seq_of(p, i, G);
            if (seq >= 0 && seq < p.n_seqs) row = seq * p.Hq + it.head_of(kvh, i, G);
        }
        // its query, into the swizzled tile (lanes without one keep what lies there: they meet nobody else's sums)
        if (row >= 0) {
            const uint4* from = reinterpret_cast<const uint4*>(q + (size_t)row * kD);
#pragma unroll
            for (int c = 0; c < kD / 8; ++c)
                *reinterpret_cast<uint4*>(q_s + (c >> 3) * kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = from[c];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sync.q_full));
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        float m_used = -INFINITY, l_run = 0.0f;
        bool ok = true;
        for (int j = 0; j < n_tiles && has_rows; ++j) {
            const uint32_t ts = tmem_s + (uint32_t)(j & 1) * kBN + lane_addr;
            ok = mbar_wait(smem_addr(&sync.s_full[j & 1]), (j >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            // the copy's keys are columns [copy * kKeys, + kKeys)
            uint32_t v[kKeys];
#pragma unroll
            for (int c = 0; c < kKeys; c += 32) tmem_ld32_nowait(ts + copy * kKeys + c, *reinterpret_cast<uint32_t(*)[32]>(&v[c]));
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kKeys; c += 32) tmem_landed(*reinterpret_cast<uint32_t(*)[32]>(&v[c]));
            const int valid = it.end - it.begin - j * kBN - copy * kKeys;
            if (valid < kKeys) {
#pragma unroll
                for (int k = 0; k < kKeys; ++k) v[k] = k < valid ? v[k] : __float_as_uint(-INFINITY);
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < kKeys; ++k) top[k & 3] = fmaxf(top[k & 3], __uint_as_float(v[k]));
            const float highest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            float f = 1.0f;
            if ((highest - m_used) * p.scale_log2 > kLazyRescale) {       // also the first keys: m_used = -inf
                f = ex2((m_used - highest) * p.scale_log2);
                m_used = highest;
                l_run *= f;
            }
            const float lower = m_used == -INFINITY ? 0.0f : -m_used * p.scale_log2;
            float l0 = 0.0f, l1 = 0.0f;
            // the weights, two a column, over the first half of S; every lane of the warp has read its scores
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < kBN / 2; c += 16) {
                if (c >= copy * kKeys / 2 && c < (copy + 1) * kKeys / 2) continue;
#pragma unroll
                for (int k = 0; k < 16; ++k) pk[k] = 0u;
                tmem_st16(ts + c, pk);
            }
#pragma unroll
            for (int c = 0; c < kKeys; c += 32) {
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float p0 = ex2(fmaf(__uint_as_float(v[c + k]), p.scale_log2, lower));
                    const float p1 = ex2(fmaf(__uint_as_float(v[c + k + 1]), p.scale_log2, lower));
                    l0 += p0;
                    l1 += p1;
                    pk[k >> 1] = pack_bf16x2(p0, p1);
                }
                tmem_st16(ts + copy * (kKeys / 2) + (c >> 1), pk);
            }
            l_run += l0 + l1;
            if (j > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
                ok = mbar_wait(smem_addr(&sync.o_full), (j - 1) & 1, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
#pragma unroll 1
                for (int c = 0; c < kD; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem_o + lane_addr + c, o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st32(tmem_o + lane_addr + c, o);
                }
            }
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sync.p_full[j & 1]));
        }
        // a thread has a row's copy, a warp writes a row: they meet in shared memory, which the products have done with
        constexpr int kPitch = kD + 4;
        float* rows = reinterpret_cast<float*>(k_s);                      // [128][kPitch]
        float4* ends = reinterpret_cast<float4*>(rows + kBM * kPitch);    // [128]: m, l, the row's number
        if (n_tiles > 0 && ok) {
            ok = mbar_wait(smem_addr(&sync.o_done), 0, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
        }
        if (has_rows) {
#pragma unroll 1
            for (int c = 0; c < kD; c += 32) {
                uint32_t o[32];
                if (n_tiles > 0) {
                    tmem_ld32(tmem_o + lane_addr + c, o);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0u;
                }
#pragma unroll
                for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4*>(rows + r * kPitch + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
            ends[r] = make_float4(m_used == -INFINITY ? m_used : m_used * p.scale_log2, l_run, __int_as_float(row), 0.0f);
        }
        meet();
        if (ok) {
            const int parts = p.n_shared + p.n_own;
            for (int k = warp; k < it.rows; k += 4) {
                float m = -INFINITY;
#pragma unroll
                for (int c = 0; c < REPEAT; ++c) m = fmaxf(m, ends[c * (kBM / REPEAT) + k].x);
                const float base = m == -INFINITY ? 0.0f : m;
                float2 a = make_float2(0.0f, 0.0f), b = a;
                float l = 0.0f;
#pragma unroll
                for (int c = 0; c < REPEAT; ++c) {
                    const int from = c * (kBM / REPEAT) + k;
                    const float f = ex2(ends[from].x - base);
                    const float2* o = reinterpret_cast<const float2*>(rows + from * kPitch);
                    const float2 x = o[lane], y = o[lane + 32];
                    a.x = fmaf(x.x, f, a.x); a.y = fmaf(x.y, f, a.y);
                    b.x = fmaf(y.x, f, b.x); b.y = fmaf(y.y, f, b.y);
                    l = fmaf(ends[from].y, f, l);
                }
                const int to = __float_as_int(ends[k].z);
                if (to < 0) continue;
                float* dst = partial + ((size_t)to * parts + it.part) * (kD + 2);
                reinterpret_cast<float2*>(dst)[lane] = a;
                reinterpret_cast<float2*>(dst)[lane + 32] = b;
                if (lane == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(m, l);
            }
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicMax(error, 4u); }
    }
    __syncwarp();
    if (*abort_flag) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);         // copies and products in flight land before the memory is reused
    }
    fence_before();
    __syncthreads();
    if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(kTmemColumns));
}

template <int REPEAT>
int launch_repeat(const void* q, const Maps& maps, float* partial, const Shared& p, cudaStream_t stream) {
    const long long blocks = family_blocks(p, p.Hq / p.Hkv, kBM / REPEAT);
    if (blocks > 0x7fffffff) return PB_ERR_TOO_LARGE;
    static SmemLimit limit;
    static DeviceLimit most;
    int rc = limit.allow(shared_tcgen05_kernel<REPEAT>, kSmemBytes);
    if (rc == 0) rc = share_most(most, shared_tcgen05_kernel<REPEAT>);
    if (rc != 0) return rc;
    shared_tcgen05_kernel<REPEAT><<<dim3((unsigned)blocks, p.Hkv), kThreads, kSmemBytes, stream>>>((const bf16*)q, maps.k, maps.v, partial, p,
                                                                                                   attn5::log2_exact(p.page_size), pool_bounds_now(), maps.error);
    return launch_status();
}

}  // namespace

namespace pb {
namespace shared_attention {

int launch_tcgen05(const void* q, const Maps& maps, float* partial, const Shared& p, cudaStream_t stream) {
    const int rows = p.most_members * (p.Hq / p.Hkv);
    if (rows <= 32) return launch_repeat<4>(q, maps, partial, p, stream);
    return rows <= 64 ? launch_repeat<2>(q, maps, partial, p, stream) : launch_repeat<1>(q, maps, partial, p, stream);
}

}  // namespace shared_attention
}  // namespace pb

// A new limit of this kernel's bounded waits in clock cycles.
PB_EXPORT int pb_shared_tcgen05_wait_limit(long long limit) {
    return limit > 0 && cudaMemcpyToSymbol(g_wait_limit, &limit, sizeof(limit)) == cudaSuccess ? 0 : -1;
}

// Lets one of these waits run out: afterwards the error word reads 9.  Set a short limit first.
namespace {
struct SharedTcgen05Unit {};
}
PB_EXPORT int pb_shared_tcgen05_wait_selftest(unsigned int* error, cudaStream_t stream) {
    if (error == nullptr) return PB_ERR_BAD_SIZE;
    wait_gives_up_kernel<SharedTcgen05Unit><<<1, 32, 0, stream>>>(error);
    return launch_status();
}
