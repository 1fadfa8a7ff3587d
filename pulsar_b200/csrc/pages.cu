// Pages of a cache copied inside its pools or into other pools: dst_pool[e, dst[i]] = src_pool[e, src[i]] for every pool, every
// entry e (layer) of it and every pair i.
//
// A page of one entry is one run of page_bytes bytes, so the copy is nothing but reads and writes: bound by memory, 2 bytes moved
// per byte copied.  All pools, entries and pairs go in one launch (a fork copies one page of each of 36 layers' keys and values: 72
// runs of 32 KB, far too little for a launch each).
//
// No page may be both read and written by one call (the pairs are not ordered).  A pair with an id outside its pool is left out.
#include "common.cuh"

namespace {

using namespace pb;

constexpr int kMaxPools = 16;
constexpr int kThreads = 128;
constexpr int kVectors = 4;                              // units in flight per thread

// The widest unit, for addresses and sizes that are multiples of 32 bytes.  FIRST: what it reads and writes is first to leave L2, as suits a
// copy that does not fit there.  (1,000 pages of 36 layers, 4.7 GB read and written, take 735 to 780 us by where the pools lie; 16 bytes a
// unit 815, whatever the threads, units and blocks 2 to 10 % more than 32, and bulk copies through shared memory no less.)
template <bool FIRST>
struct alignas(32) Wide {
    uint32_t word[8];
};
template <typename T> __device__ __forceinline__ T load_unit(const T* p) { return *p; }
template <typename T> __device__ __forceinline__ void store_unit(T* p, const T& v) { *p = v; }
template <bool FIRST> __device__ __forceinline__ Wide<FIRST> load_unit(const Wide<FIRST>* p) {
    Wide<FIRST> v;
    if (FIRST)
        asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v.word[0]), "=r"(v.word[1]), "=r"(v.word[2]), "=r"(v.word[3]), "=r"(v.word[4]), "=r"(v.word[5]), "=r"(v.word[6]), "=r"(v.word[7])
                     : "l"(p));
    else
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v.word[0]), "=r"(v.word[1]), "=r"(v.word[2]), "=r"(v.word[3]), "=r"(v.word[4]), "=r"(v.word[5]), "=r"(v.word[6]), "=r"(v.word[7])
                     : "l"(p));
    return v;
}
template <bool FIRST> __device__ __forceinline__ void store_unit(Wide<FIRST>* p, const Wide<FIRST>& v) {
    if (FIRST)
        asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "r"(v.word[0]), "r"(v.word[1]), "r"(v.word[2]), "r"(v.word[3]), "r"(v.word[4]), "r"(v.word[5]), "r"(v.word[6]), "r"(v.word[7]) : "memory");
    else
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "r"(v.word[0]), "r"(v.word[1]), "r"(v.word[2]), "r"(v.word[3]), "r"(v.word[4]), "r"(v.word[5]), "r"(v.word[6]), "r"(v.word[7]) : "memory");
}

struct PoolCopy {
    const unsigned char* src;
    unsigned char* dst;
    long long src_entry, dst_entry;                      // bytes from an entry to the next
    long long page_bytes;
    int src_pages, dst_pages;
    unsigned int first;                                  // chunks of the pools before this one
    unsigned int chunks;                                 // chunks per page
};
struct Pools {
    PoolCopy pool[kMaxPools];
    int n;
    unsigned int total;                                  // chunks of all pools (a terabyte has 2^26 of them)
};

// One chunk of a page per block and turn, in units of T.
template <typename T>
__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(const __grid_constant__ Pools pools, const int* __restrict__ src, const int* __restrict__ dst, unsigned int n_pairs) {
    constexpr int kChunk = kThreads * kVectors;          // units
    for (unsigned int work = blockIdx.x; work < pools.total; work += gridDim.x) {
        int k = 0;
        while (k + 1 < pools.n && work >= pools.pool[k + 1].first) ++k;
        const PoolCopy& p = pools.pool[k];
        const unsigned int run = (work - p.first) / p.chunks, chunk = work - p.first - run * p.chunks;
        const unsigned int entry = run / n_pairs, pair = run - entry * n_pairs;
        const int from = src[pair], to = dst[pair];
        if (from < 0 || from >= p.src_pages || to < 0 || to >= p.dst_pages) continue;
        const T* a = reinterpret_cast<const T*>(p.src + entry * p.src_entry + (long long)from * p.page_bytes) + (long long)chunk * kChunk;
        T* b = reinterpret_cast<T*>(p.dst + entry * p.dst_entry + (long long)to * p.page_bytes) + (long long)chunk * kChunk;
        const long long left = p.page_bytes / (long long)sizeof(T) - (long long)chunk * kChunk;
        T v[kVectors];
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
            if (threadIdx.x + i * kThreads < left) v[i] = load_unit(a + threadIdx.x + i * kThreads);
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
            if (threadIdx.x + i * kThreads < left) store_unit(b + threadIdx.x + i * kThreads, v[i]);
    }
}

template <typename T>
int launch(Pools& pools, const int* src, const int* dst, int n_pairs, const int* entries, cudaStream_t stream) {
    long long first = 0;
    for (int k = 0; k < pools.n; ++k) {
        PoolCopy& p = pools.pool[k];
        const long long units = p.page_bytes / (long long)sizeof(T);
        const long long chunks = (units + kThreads * kVectors - 1) / (kThreads * kVectors);
        if (chunks > 0x7fffffff) return PB_ERR_TOO_LARGE;
        p.chunks = (unsigned int)chunks;
        p.first = (unsigned int)first;
        if (chunks * entries[k] > 0x7fffffff / n_pairs) return PB_ERR_TOO_LARGE;
        first += chunks * entries[k] * n_pairs;
    }
    if (first > 0x7fffffff) return PB_ERR_TOO_LARGE;
    pools.total = (unsigned int)first;
    const long long most = 148 * 16;
    copy_pages_kernel<T><<<(int)(first < most ? first : most), kThreads, 0, stream>>>(pools, src, dst, (unsigned int)n_pairs);
    return launch_status();
}

}  // namespace

// `pools` pools of at most 16, described by six numbers each in `shapes`: bytes from an entry to the next in the source and in the
// destination, bytes of a page, pages of the source and of the destination, entries.  src, dst: int32 [n_pairs] on the device.
PB_EXPORT int pb_copy_pages(int n_pools, const void* const* from, void* const* to, const long long* shapes, const int* src, const int* dst,
                            int n_pairs, cudaStream_t stream) {
    if (n_pools < 0 || n_pairs < 0) return PB_ERR_BAD_SIZE;
    if (n_pools > kMaxPools) return PB_ERR_TOO_LARGE;
    Pools pools = {};
    int entries[kMaxPools];
    unsigned long long bits = 0;
    for (int i = 0; i < n_pools; ++i) {
        const long long* s = shapes + 6 * i;
        if (s[2] < 0 || s[3] < 0 || s[4] < 0 || s[5] < 0 || s[3] > 0x7fffffff || s[4] > 0x7fffffff || s[5] > 0x7fffffff) return PB_ERR_BAD_SIZE;
        if (s[2] == 0 || s[5] == 0) continue;            // nothing in it
        PoolCopy& p = pools.pool[pools.n];
        p.src = static_cast<const unsigned char*>(from[i]);
        p.dst = static_cast<unsigned char*>(to[i]);
        p.src_entry = s[0]; p.dst_entry = s[1]; p.page_bytes = s[2]; p.src_pages = (int)s[3]; p.dst_pages = (int)s[4];
        entries[pools.n++] = (int)s[5];
        bits |= (unsigned long long)p.src | (unsigned long long)p.dst | (unsigned long long)s[0] | (unsigned long long)s[1] | (unsigned long long)s[2];
    }
    if (pools.n == 0 || n_pairs == 0) return 0;
    // the widest unit that every address and size is a multiple of
    if ((bits & 31) == 0) {
        long long moved = 0;                             // a pool's entries x pairs x bytes, read and written
        for (int k = 0; k < pools.n; ++k) moved += 2 * pools.pool[k].page_bytes * entries[k] * n_pairs;
        return moved > 96LL << 20 ? launch<Wide<true>>(pools, src, dst, n_pairs, entries, stream) : launch<Wide<false>>(pools, src, dst, n_pairs, entries, stream);
    }
    if ((bits & 15) == 0) return launch<uint4>(pools, src, dst, n_pairs, entries, stream);
    if ((bits & 3) == 0) return launch<uint32_t>(pools, src, dst, n_pairs, entries, stream);
    return launch<unsigned char>(pools, src, dst, n_pairs, entries, stream);
}
