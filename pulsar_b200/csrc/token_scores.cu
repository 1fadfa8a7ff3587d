// What rows of logits say of given tokens: log probability, rank, the row's entropy and its likeliest tokens.
//
// One pass over the row: every thread keeps the maximum and the sums (scores.cuh) of what it has seen, and counts the logits beyond the
// given token's.  Bound by the bytes of the logits where there are rows enough, by latency where there are few: a row is cut among the
// blocks of a cluster (up to eight), whose results meet in the first block's hands through distributed shared memory, so there is one
// launch, no scratch memory and no order of atomics that a result could depend on.  (float32, us, without and with 8 alternatives: 2 rows of
// 151,936 8 and 11, 64 rows 14 and 17, 2,000 rows 197 and 266, where the bytes take 188; 2,000 rows of 32,000 49 and 74, bytes 40.  bfloat16
// is bound by instructions: 2,000 rows of 151,936 with 8 take 170, bytes 94, with 12.5 instructions a logit, which fill the schedulers' issue slots
// to 65 %; 777 rows of 32,003 take 15.6 a logit and 25 us, one round of blocks whose selection no other block's pass hides.)
//
// The n likeliest (n <= 32) cost the pass nothing but the number of the chunk in which a thread's maximum rose last.  A key of 64 bits
// holds a logit's bits, made to compare as unsigned numbers, above the complement of its index: of equal logits the lower index is the larger
// key, and no two keys are equal.  The n-th largest of the thread groups' largest keys is reached by n keys at least, so no key below it is
// among the n likeliest, and only the few threads whose own largest reaches it can hold any that are: their elements are read once more (some 5
// to 10 % of the row, but 16 bytes here and there: memory brings a quarter of 200 float32 rows again, 46 % of 2,000 bfloat16 ones, with 128
// threads a row; rows that fit L2 come from there), what reaches the threshold is ranked by counting.  Should more than kMostCandidates reach it (a row made
// so that few threads hold all its large logits), the likeliest are found one by one.  In the order of tokens a NaN is below every
// number; a thread that met one is always read again.
#include "scores.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

using namespace pb;

constexpr int kMostThreads = 512;
constexpr int kMostWarps = kMostThreads / 32;
constexpr int kGroups = 64;                  // of neighbouring threads, whose largest keys are compared
constexpr int kMostCandidates = 1024;
constexpr int kMostCluster = 8;              // the portable limit
constexpr int kMostTop = 32;

typedef unsigned long long Key;

__device__ __forceinline__ Key key_of(float x, int index) {
    const uint32_t bits = __float_as_uint(x + 0.0f);                          // -0 is +0
    const uint32_t up = x != x ? 0u : (bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u));
    return ((Key)up << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float logit_of(Key k) {
    const uint32_t up = (uint32_t)(k >> 32);
    return up == 0 ? nanf("") : __uint_as_float((up >> 31) ? up ^ 0x80000000u : ~up);
}

// 16 bytes of a row as float32.
template <typename T> constexpr int kPerVector = 16 / (int)sizeof(T);
__device__ __forceinline__ void widen(const uint4& u, const float*, float* x) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void widen(const uint4& u, const __nv_bfloat16*, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 load_once(const uint4* p) {                  // (a row is read once: it need not stay in L1)
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A chunk of sixteen logits joins the sums.
__device__ __forceinline__ void add_chunk(Stats& st, const uint4 (&v)[4], const float* tag) {
    float x[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) widen(v[j], tag, x + 4 * j);
    add_logits(st, x);
}
// bfloat16: the maximum, and the bound that keeps differences finite, are found on pairs as they are (half the instructions, which is what
// a row of bfloat16 is bound by).  The bound is 1,000 below the maximum, or a 64th of it, which is more than bfloat16's step, and is rounded
// down: no number that weighs anything is raised to it.
__device__ __forceinline__ void add_chunk(Stats& st, const uint4 (&v)[2], const __nv_bfloat16* tag) {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    __nv_bfloat162 pair[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pair[i] = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
    const __nv_bfloat162 high = __hmax2(__hmax2(__hmax2(pair[0], pair[1]), __hmax2(pair[2], pair[3])),
                                        __hmax2(__hmax2(pair[4], pair[5]), __hmax2(pair[6], pair[7])));
    raise(st, fmaxf(__low2float(high), __high2float(high)));
    if (st.m < -1e38f && st.m > -INFINITY) {             // there is no room below such a maximum for the bound
        float x[16];
        widen(v[0], tag, x);
        widen(v[1], tag, x + 8);
        add_logits(st, x);
        return;
    }
    const float base = st.m == -INFINITY ? 0.0f : st.m;
    const __nv_bfloat162 bound = __bfloat162bfloat162(__float2bfloat16_rd(base - fmaxf(-kFar, fabsf(base) * 0.015625f)));
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 up = __hmax2_nan(pair[i], bound);
        x[2 * i] = __low2float(up);
        x[2 * i + 1] = __high2float(up);
    }
    add_bounded(st, base, x);
}

// Counts the logits of a chunk that are not below a bar of their vector's (NaN: none is counted), in ones and zeros of the logits' own type,
// two an instruction.  float32 counts a thread's whole share (below 2^24), bfloat16 a chunk (below 2^8): exact.
struct Count32 {
    Two n = 0;
    __device__ __forceinline__ void add(const uint4& v, float bar) {
        float x[4], one[4];
        widen(v, (const float*)nullptr, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(one[i]) : "f"(x[i]), "f"(bar));
        n = add2(n, add2(two(one[0], one[1]), two(one[2], one[3])));
    }
    __device__ __forceinline__ void end_chunk() {}
    __device__ __forceinline__ int total() const {
        float a, b;
        apart(n, a, b);
        return (int)a + (int)b;
    }
};
struct Count16 {
    __nv_bfloat162 n = __float2bfloat162_rn(0.0f);
    int sum = 0;
    __device__ __forceinline__ void add(const uint4& v, float bar) {
        const __nv_bfloat162 at = __float2bfloat162_rn(bar);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) n = __hadd2(n, __hge2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), at));
    }
    __device__ __forceinline__ void end_chunk() {
        sum += (int)(__low2float(n) + __high2float(n));
        n = __float2bfloat162_rn(0.0f);
    }
    __device__ __forceinline__ int total() const { return sum; }
};
template <typename T> struct CountOf { typedef Count32 type; };
template <> struct CountOf<__nv_bfloat16> { typedef Count16 type; };
// The next larger number of the logits' type (NaN behind +inf and NaN): what a logit has to reach to be beyond x.
__device__ __forceinline__ float next_up(float x, const float*) {
    if (x != x) return x;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return __uint_as_float(x == 0.0f ? 1u : (b >> 31) ? b - 1 : b + 1);
}
__device__ __forceinline__ float next_up(float x, const __nv_bfloat16*) {
    if (x != x) return x;
    const uint32_t b = __float_as_uint(x + 0.0f) >> 16;
    return __uint_as_float((x == 0.0f ? 1u : (b >> 15) ? b - 1 : b + 1) << 16);
}
// A vector of logits that are not there.
__device__ __forceinline__ uint4 nothing(const float*) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 nothing(const __nv_bfloat16*) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

struct Scores {
    const void* logits;
    long long row_stride;
    const int* tokens;
    float *logprob, *entropy, *top_logprob;
    int *rank, *top_ids;
    int vocab, n_top;
};

// What a block hands to the first of its cluster.
struct Result {
    Stats st;
    int likelier;
    Key keys[kMostTop];
};

// The row as 16-byte vectors, with the elements in front of the first whole one and behind the last; this block's are [begin, end).
template <typename T>
struct Slice {
    const T* row;
    const uint4* vectors;
    int before, behind, first_behind;        // odd elements: [0, before) and [first_behind, first_behind + behind)
    int begin, end;
    bool odd;                                // whether the odd elements are this block's

    __device__ __forceinline__ Slice(const Scores& p, long long r, int block, int blocks) {
        constexpr int N = kPerVector<T>;
        row = static_cast<const T*>(p.logits) + r * p.row_stride;
        before = min(p.vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
        const int n = (p.vocab - before) / N;
        vectors = reinterpret_cast<const uint4*>(row + before);
        first_behind = before + n * N;
        behind = p.vocab - first_behind;
        const int each = ((n + blocks - 1) / blocks + 31) & ~31;
        begin = min(n, block * each);
        end = min(n, begin + each);
        odd = block == 0;
    }
    // the index of a vector's first element
    __device__ __forceinline__ int index(int vector) const { return before + vector * kPerVector<T>; }
    // the lane's odd element, or -1
    __device__ __forceinline__ int odd_index(int lane) const {
        if (!odd) return -1;
        return lane < before ? lane : lane - before < behind ? first_behind + lane - before : -1;
    }
};

// Registers for as many blocks on an SM as the launch counts on: one of 512 threads, two of 256, six of 128.
template <typename T, bool RANK, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 1 : THREADS == 256 ? 2 : 6)
token_scores_kernel(const Scores p) {
    constexpr int N = kPerVector<T>, V = 16 / N;                              // elements of a vector, vectors of a thread's chunk of sixteen
    __shared__ Result result;
    __shared__ Stats stats_s[kMostWarps];
    __shared__ int count_s[kMostWarps];
    __shared__ __align__(16) Key keys_s[kMostCandidates];                                  // the groups' largest, then the candidates
    __shared__ unsigned short hot_s[THREADS];
    __shared__ Key threshold_s, best_s[kMostWarps];
    __shared__ int n_hot_s, n_candidates_s;

    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = cluster.num_blocks(), block = cluster.block_rank();
    const long long r = blockIdx.x / blocks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int warps = THREADS / 32;
    const Slice<T> slice(p, r, block, blocks);
    const int step = warps * 32 * V;                                          // vectors of a turn of the whole block
    const int my_first = slice.begin + warp * 32 * V + lane;                  // + turn * step + j * 32

    uint4 next[2][V];                                                         // the next two chunks are on their way
    auto fetch = [&](uint4 (&into)[V], int first) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j * 32 < slice.end) into[j] = load_once(slice.vectors + first + j * 32);
    };
    fetch(next[0], my_first);
    fetch(next[1], my_first + step);
    const int odd_index = warp == 0 ? slice.odd_index(lane) : -1;
    const float odd_logit = odd_index >= 0 ? to_float(slice.row[odd_index]) : 0.0f;
    const int token = p.tokens[r];
    const bool known = token >= 0 && token < p.vocab;
    const float given = known ? to_float(slice.row[token]) : 0.0f;

    const float beyond = next_up(given, slice.row);
    // the first element of the vector that holds the given token (an odd element in front of all: 0, behind all: the first of those)
    const int token_vector = token < slice.before ? 0 : token >= slice.first_behind ? slice.first_behind : token - (token - slice.before) % N;

    Stats st = {-INFINITY, 0.0f, 0.0f};
    typename CountOf<T>::type beaten;
    int risen = my_first;
    auto take = [&](uint4 (&now)[V], int first) {
        const bool whole = first - lane + 32 * V <= slice.end;                // the warp's chunk ends inside the slice
        uint4 v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = !whole && first + j * 32 >= slice.end ? nothing(slice.row) : now[j];
        fetch(now, first + 2 * step);
        const float before = st.m;
        add_chunk(st, v, slice.row);
        if (RANK) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int vector = first + j * 32;
                // in front of the given token's vector equal logits count too
                const float bar = slice.index(vector) < token_vector ? given : beyond;
                beaten.add(v[j], !whole && vector >= slice.end ? nanf("") : bar);
            }
            beaten.end_chunk();
        }
        if (st.m > before) risen = first;
    };
    for (int first = my_first; first - lane < slice.end; first += 2 * step) {
        take(next[0], first);
        if (first - lane + step < slice.end) take(next[1], first + step);
    }
    const bool met_nan = st.s != st.s;
    const float highest = st.m;                                               // of this thread's chunks
    uint4 last[V];                                                            // the chunk where it rose last, for the likeliest (asked for ahead of the sums)
    if (p.n_top > 0) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (risen + j * 32 < slice.end) last[j] = slice.vectors[risen + j * 32];
    }
    int likelier = beaten.total();
    // logits equal to the given token's that stand in front of it in its own vector
    if (RANK && block == 0 && warp == warps - 1 && token_vector + lane < token && token >= slice.before && token < slice.first_behind)
        likelier += to_float(slice.row[token_vector + lane]) == given ? 1 : 0;
    Stats odd = {-INFINITY, 0.0f, 0.0f};
    if (odd_index >= 0) {
        odd = one_logit(odd_logit);
        if (RANK) likelier += odd_logit > given || (odd_logit == given && odd_index < token) ? 1 : 0;
    }
    st = warp_join(warp == 0 ? join(st, odd) : st);
    if (RANK) likelier = __reduce_add_sync(0xffffffffu, likelier);
    if (lane == 0) { stats_s[warp] = st; count_s[warp] = likelier; }

    if (p.n_top > 0) {
        // the groups' largest keys: a thread's is its highest logit's first place in the chunk where the maximum rose last
        Key key = 0;
#pragma unroll
        for (int j = V - 1; j >= 0; --j) {
            const int vector = risen + j * 32;
            if (vector < slice.end) {
                float x[N];
                widen(last[j], slice.row, x);
#pragma unroll
                for (int i = N - 1; i >= 0; --i)
                    if (x[i] == highest) key = (Key)(slice.index(vector) + i + 1);
            }
        }
        if (key != 0) key = key_of(highest, (int)key - 1);
        const Key own = key;
        constexpr int per_group = THREADS / kGroups;
#pragma unroll
        for (int o = 1; o < per_group; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        const bool speaks = tid % per_group == 0;
        const int group = tid / per_group;
        if (tid == 0) { threshold_s = 0; n_hot_s = 0; n_candidates_s = 0; }
        if (tid < kMostTop) result.keys[tid] = 0;
        if (speaks) keys_s[group] = key;
        __syncthreads();
        {
            // the threads of a group share its comparisons
            const Key mine = keys_s[group];
            int larger = 0;
#pragma unroll 4
            for (int g = 2 * (tid % per_group); g < kGroups; g += 2 * per_group) {
                const ulonglong2 some = *reinterpret_cast<const ulonglong2*>(keys_s + g);
                larger += (some.x > mine ? 1 : 0) + (some.y > mine ? 1 : 0);
            }
            for (int o = 1; o < per_group; o <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
            if (speaks && mine != 0 && larger == p.n_top - 1) threshold_s = mine;
        }
        __syncthreads();
        const Key threshold = threshold_s;                                    // 0: fewer groups have elements than are asked for
        if ((own != 0 && own >= threshold) || met_nan) hot_s[atomicAdd(&n_hot_s, 1)] = (unsigned short)tid;
        __syncthreads();
        const int turns = (slice.end - slice.begin + step - 1) / step;
        const float threshold_logit = logit_of(threshold);                    // (NaN where there is no threshold: then no logit is below it)
        auto candidate = [&](float x, int index) {
            if (x < threshold_logit) return;
            const Key k = key_of(x, index);
            if (k >= threshold) {
                const int at = atomicAdd(&n_candidates_s, 1);                 // (ranked below: their order here does not matter)
                if (at < kMostCandidates) keys_s[at] = k;
            }
        };
        // the hot threads' vectors, all of them side by side; a thread asks for four before it looks at one
        const int of_one = turns * V, of_all = n_hot_s * of_one;
        const float share = 1.0f / of_one;                                    // (item + 1/2) share has the whole part of item / of_one below 2^20 items
        for (int item0 = tid; item0 < of_all; item0 += 4 * THREADS) {
            uint4 v[4];
            int at[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int item = item0 + u * THREADS;
                at[u] = slice.end;
                if (item < of_all) {
                    const int h = of_all < (1 << 20) ? (int)((item + 0.5f) * share) : item / of_one, q = item - h * of_one;
                    const int owner = hot_s[h];
                    at[u] = slice.begin + (owner >> 5) * 32 * V + (owner & 31) + q / V * step + q % V * 32;
                    if (at[u] < slice.end) v[u] = slice.vectors[at[u]];
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (at[u] < slice.end) {
                    float x[N];
                    widen(v[u], slice.row, x);
#pragma unroll
                    for (int i = 0; i < N; ++i) candidate(x[i], slice.index(at[u]) + i);
                }
            }
        }
        if (odd_index >= 0) candidate(odd_logit, odd_index);
        __syncthreads();
        const int n = n_candidates_s;
        if (n <= kMostCandidates) {
            for (int i = tid; i < n; i += THREADS) {
                const Key mine = keys_s[i];
                int larger = 0;
#pragma unroll 4
                for (int g = 0; g < n; ++g) larger += keys_s[g] > mine ? 1 : 0;
                if (larger < p.n_top) result.keys[larger] = mine;
            }
        } else {
            Key below = ~(Key)0;
            for (int i = 0; i < p.n_top && below != 0; ++i) {
                Key best = 0;
                for (int vector = slice.begin + tid; vector < slice.end; vector += THREADS) {
                    float x[N];
                    widen(slice.vectors[vector], slice.row, x);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const Key k = key_of(x[e], slice.index(vector) + e);
                        if (k < below) best = max(best, k);
                    }
                }
                if (odd_index >= 0) {
                    const Key k = key_of(odd_logit, odd_index);
                    if (k < below) best = max(best, k);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
                __syncthreads();
                if (lane == 0) best_s[warp] = best;
                __syncthreads();
                below = 0;
                for (int w = 0; w < warps; ++w) below = max(below, best_s[w]);
                if (tid == 0) result.keys[i] = below;
            }
        }
    }
    __syncthreads();
    if (warp == 0) {
        st = warp_join(lane < warps ? stats_s[lane] : Stats{-INFINITY, 0.0f, 0.0f});
        likelier = __reduce_add_sync(0xffffffffu, lane < warps ? count_s[lane] : 0);
        if (lane == 0) { result.st = st; result.likelier = likelier; }
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    if (block == 0) {
        if (warp == 0) {
            st = warp_join(lane < blocks ? cluster.map_shared_rank(&result, lane)->st : Stats{-INFINITY, 0.0f, 0.0f});
            likelier = __reduce_add_sync(0xffffffffu, lane < blocks ? cluster.map_shared_rank(&result, lane)->likelier : 0);
            if (lane == 0) stats_s[0] = Stats{st.m, logf(st.s), st.t / st.s};
        } else {
            for (int i = tid - 32; i < blocks * p.n_top; i += THREADS - 32)
                keys_s[i] = cluster.map_shared_rank(&result, i / p.n_top)->keys[i % p.n_top];
        }
        __syncthreads();
        if (blocks > 1) cluster.barrier_arrive();                             // the others' results are here: they may leave
        const float m = stats_s[0].m, log_s = stats_s[0].s;
        if (tid == 0) {
            p.logprob[r] = known ? (given - m) - log_s : nanf("");
            p.entropy[r] = log_s - stats_s[0].t;
            if (RANK) p.rank[r] = known ? likelier : -1;
        }
        for (int i = tid; i < blocks * p.n_top; i += THREADS) {
            const Key mine = keys_s[i];
            int larger = i;                                                   // its own block's keys are in order
            if (blocks > 1) {                                                 // and so are the others': searched all at once
                int more[kMostCluster] = {};
#pragma unroll
                for (int jump = kMostTop; jump > 0; jump >>= 1)
#pragma unroll
                    for (int b = 0; b < kMostCluster; ++b)
                        if (b < blocks && more[b] + jump <= p.n_top && keys_s[b * p.n_top + more[b] + jump - 1] > mine) more[b] += jump;
                larger = 0;
#pragma unroll
                for (int b = 0; b < kMostCluster; ++b) larger += more[b];
            }
            if (mine != 0 && larger < p.n_top) {
                p.top_ids[r * p.n_top + larger] = index_of(mine);
                p.top_logprob[r * p.n_top + larger] = (logit_of(mine) - m) - log_s;
            }
        }
    }
    if (blocks > 1) {                                                         // no block leaves while the first still reads its result
        if (block != 0) cluster.barrier_arrive();
        cluster.barrier_wait();
    }
}

template <typename T, bool RANK, int THREADS>
int launch(const Scores& p, int rows, int cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * cluster);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, token_scores_kernel<T, RANK, THREADS>, p);
}

template <typename T, bool RANK>
int launch(const Scores& p, int rows, cudaStream_t stream) {
    // What follows the pass over a row costs every block of it the same work: so no more blocks than two of 256 threads an SM, none with
    // less than 4,096 logits.  (64 rows of 151,936 float32 with 8 alternatives, blocks a row x threads: 4 x 256 17 us, 1 x 512 19, 8 x 128 20;
    // beyond two blocks an SM small ones hide each other's ends: 2,000 rows of 32,000 with 8 alternatives, 128 threads 74 us, 256 82, 512 117.)
    int cluster = 1;
    while (cluster < kMostCluster && (long long)rows * cluster * 2 <= 2 * 148 && p.vocab / (cluster * 2) >= 4096) cluster *= 2;
    const long long blocks = (long long)rows * cluster;
    if (blocks > 0x7fffffff) return PB_ERR_TOO_LARGE;
    if (blocks <= 148) return launch<T, RANK, 512>(p, rows, cluster, stream);
    // The elements of a thread in n_top are read once more: of more threads that is a smaller share, which pays where a row is long and its
    // elements are four bytes (500 rows of 100,352 with 8 alternatives: 51 against 59 us, of 64,000: 39 against 41, of 32,000: 27 against
    // 25; 2,000 rows of 151,936 bfloat16: 200 against 170).
    if (blocks <= 2 * 148 || (sizeof(T) == 4 && p.n_top > 0 && p.vocab >= 65536)) return launch<T, RANK, 256>(p, rows, cluster, stream);
    return launch<T, RANK, 128>(p, rows, cluster, stream);
}

}  // namespace

// logits [rows, vocab] (dtype 0 float32, 1 bfloat16), row_stride elements from a row to the next; tokens, rank, top_ids int32, the other
// results float32; rank may be null, top_ids and top_logprob [rows, n_top] are null where n_top is 0 (n_top <= 32, <= vocab).
PB_EXPORT int pb_token_scores(int dtype, const void* logits, long row_stride, int rows, int vocab, const int* tokens, float* logprob, float* entropy,
                              int* rank, int* top_ids, float* top_logprob, int n_top, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (dtype != PB_F32 && dtype != PB_BF16) return PB_ERR_BAD_DTYPE;
    if (vocab <= 0 || n_top < 0 || n_top > kMostTop || n_top > vocab || row_stride < 0) return PB_ERR_BAD_SIZE;
    if (n_top > 0 && (top_ids == nullptr || top_logprob == nullptr)) return PB_ERR_BAD_SIZE;
    const Scores p = {logits, row_stride, tokens, logprob, entropy, top_logprob, rank, top_ids, vocab, n_top};
    if (dtype == PB_F32) return rank != nullptr ? launch<float, true>(p, rows, stream) : launch<float, false>(p, rows, stream);
    return rank != nullptr ? launch<__nv_bfloat16, true>(p, rows, stream) : launch<__nv_bfloat16, false>(p, rows, stream);
}
