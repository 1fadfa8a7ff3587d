// The shared sides of the attention over a forked cache (attention_shared.cu) on the fifth-generation tensor cores: bfloat16, head size 128,
// pages of 8, 16, 32 or 64 keys.
//
// A block has up to 128 query rows of a family (members x the group's heads) and one split of the family's shared keys.  The rows are the
// lanes of tensor memory: S = Q K^T (tcgen05.mma, 128 x 128 x 16 steps, operands in shared memory), a thread per row takes its row of S,
// keeps maximum and sum in float32 and writes P = 2^(s c - m c), rounded to bfloat16, over S; O += P V reads P from tensor memory and V as it
// lies in the pages.  The product costs the same for one row as for 128, so a key tile passes the tensor cores once however many of the
// family's sequences there are: bound by the bytes of the keys and values.  (mma.sync takes 2,100 cycles for 32 rows x 64 keys, with two
// blocks an SM as long as the bytes do, and so many times that for larger families.)
//
// Roles: warps 0-3 softmax (and the gathering of the query rows, which lie with their sequences), warp 4 issues the products, warp 5 brings K
// and warp 6 V, a lane per half page.  S has two buffers, S of the next tile is issued before O += P V of this one.  The maximum moves only
// when it grew by more than 2^8; O is rescaled in tensor memory only then, and the sums use the same maximum.
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
constexpr int kStages = 2;                       // K tiles, and V tiles, on their way: what is left of an SM takes a block of the own sides' kernel
constexpr int kSmemBytes = (1 + 2 * kStages) * kTileBytes + 1024;
constexpr int kTmemColumns = 512;                // S[0] | S[1] | O, and what is left of a power of two

struct Sync {
    uint64_t q_full, o_full, o_done, s_full[2], p_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint32_t tmem;
    int gave_up;
};

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
    Item it;
    if (!family_item<kBM, kBN>(p, blockIdx.x, G, it)) return;
    const int n_tiles = it.begin < it.end ? (it.end - it.begin + kBN - 1) / kBN : 0;          // (a split begins at a multiple of kBN)
    const int active = (it.rows + 31) / 32;      // softmax warps that have rows
    volatile int* abort_flag = &sync.gave_up;

    if (tid == 128) {
        mbar_init(smem_addr(&sync.q_full), 4);
        mbar_init(smem_addr(&sync.o_full), 1);
        mbar_init(smem_addr(&sync.o_done), 1);
        for (int i = 0; i < 2; ++i) { mbar_init(smem_addr(&sync.s_full[i]), 1); mbar_init(smem_addr(&sync.p_full[i]), active); }
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
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sync.tmem)), "r"(kTmemColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
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
        // ---------------- softmax: thread r owns query row r
        const int r = warp * 32 + lane;
        long long row = -1;                                       // sequence * Hq + head
        if (r < it.rows) {
            const int seq = it.seq_of(p, r, G);
            if (seq >= 0 && seq < p.n_seqs) row = (long long)seq * p.Hq + it.head_of(kvh, r, G);
        }
        // its query, into the swizzled tile (rows without one stay what they are: they meet nobody else's sums)
        if (row >= 0) {
            const uint4* from = reinterpret_cast<const uint4*>(q + row * kD);
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
        for (int j = 0; j < n_tiles && warp < active; ++j) {
            const uint32_t ts = tmem_s + (uint32_t)(j & 1) * kBN + lane_addr;
            ok = mbar_wait(smem_addr(&sync.s_full[j & 1]), (j >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            uint32_t v[kBN];
#pragma unroll
            for (int c = 0; c < kBN; c += 32) tmem_ld32_nowait(ts + c, *reinterpret_cast<uint32_t(*)[32]>(&v[c]));
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kBN; c += 32) tmem_landed(*reinterpret_cast<uint32_t(*)[32]>(&v[c]));
            const int valid = it.end - it.begin - j * kBN;
            if (valid < kBN) {
#pragma unroll
                for (int i = 0; i < kBN; ++i) v[i] = i < valid ? v[i] : __float_as_uint(-INFINITY);
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kBN; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[i]));
            const float highest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            float f = 1.0f;
            if ((highest - m_used) * p.scale_log2 > kLazyRescale) {       // also the first keys: m_used = -inf
                f = ex2((m_used - highest) * p.scale_log2);
                m_used = highest;
                l_run *= f;
            }
            const float lower = m_used == -INFINITY ? 0.0f : -m_used * p.scale_log2;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int c = 0; c < kBN; c += 32) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float p0 = ex2(fmaf(__uint_as_float(v[c + i]), p.scale_log2, lower));
                    const float p1 = ex2(fmaf(__uint_as_float(v[c + i + 1]), p.scale_log2, lower));
                    l0 += p0;
                    l1 += p1;
                    pk[i >> 1] = pack_bf16x2(p0, p1);
                }
                tmem_st16(ts + (c >> 1), pk);
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
        if (ok && warp < active) {
            const int parts = p.n_shared + p.n_own;
            // a thread has a row, a warp writes a row: they change places in shared memory, which the products have done with
            constexpr int kPitch = kD + 4;
            float* rows = reinterpret_cast<float*>(k_s) + warp * 32 * kPitch;
            if (n_tiles > 0) {
                ok = mbar_wait(smem_addr(&sync.o_done), 0, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                fence_after();
            }
            if (ok) {
#pragma unroll 1
                for (int c = 0; c < kD; c += 32) {
                    uint32_t o[32];
                    if (n_tiles > 0) {
                        tmem_ld32(tmem_o + lane_addr + c, o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(rows + lane * kPitch + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
                __syncwarp();
                const float m_log2 = m_used == -INFINITY ? m_used : m_used * p.scale_log2;
                for (int i = 0; i < 32; ++i) {
                    const long long to = __shfl_sync(0xffffffffu, row, i);
                    const float m = __shfl_sync(0xffffffffu, m_log2, i), l = __shfl_sync(0xffffffffu, l_run, i);
                    if (to < 0) continue;
                    float* dst = partial + (to * parts + it.part) * (kD + 2);
                    const float2* from = reinterpret_cast<const float2*>(rows + i * kPitch);
                    reinterpret_cast<float2*>(dst)[lane] = from[lane];
                    reinterpret_cast<float2*>(dst)[lane + 32] = from[lane + 32];
                    if (lane == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(m, l);
                }
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

}  // namespace

namespace pb {
namespace shared_attention {

int launch_tcgen05(const void* q, const Maps& maps, float* partial, const Shared& p, cudaStream_t stream) {
    const long long blocks = family_blocks(p, p.Hq / p.Hkv, kTcgen05Rows);
    if (blocks > 0x7fffffff) return PB_ERR_TOO_LARGE;
    static SmemLimit limit;
    static DeviceLimit most;
    int rc = limit.allow(shared_tcgen05_kernel, kSmemBytes);
    if (rc == 0) rc = share_most(most, shared_tcgen05_kernel);
    if (rc != 0) return rc;
    shared_tcgen05_kernel<<<dim3((unsigned)blocks, p.Hkv), kThreads, kSmemBytes, stream>>>((const bf16*)q, maps.k, maps.v, partial, p, attn5::log2_exact(p.page_size),
                                                                                           pool_bounds_now(), maps.error);
    return launch_status();
}

}  // namespace shared_attention
}  // namespace pb

// A new limit of this kernel's bounded waits in clock cycles.
PB_EXPORT int pb_shared_tcgen05_wait_limit(long long limit) {
    return limit > 0 && cudaMemcpyToSymbol(g_wait_limit, &limit, sizeof(limit)) == cudaSuccess ? 0 : -1;
}
