// What the kernels of the attention over shared pages have in common: the call's arrays, and the piece of work that a block finds in them.
#pragma once

#include "common.cuh"

#include <cuda.h>

namespace pb {
namespace shared_attention {

// 2^x by the special-function unit alone, 2 ulp as exp2f has them; results below 2^-126 are 0.
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Shared {
    const int* block_table;
    const int* kv_len;          // [n_seqs]
    const int* shared_len;      // [n_seqs]: keys [0, shared_len) are read with the family; 0: no family
    const int* members;         // the families' sequences, one family behind the other
    const int* family_start;    // [n_families + 1]
    int n_seqs, n_members, n_families, most_members;
    int table_stride;
    int Hq, Hkv, page_size;
    int n_shared, n_own;        // parts that a row has room for, of either side
    int own_chunk;              // keys of a part of a sequence's own, a multiple of the tiles
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

// A family's shared keys in at most n_shared parts of whole tiles: the keys of a part, and how many parts they make (short families fewer).
__device__ __forceinline__ int shared_keys(const Shared& p, int seq) { return max(0, min(p.shared_len[seq], p.table_stride * p.page_size)); }
__device__ __forceinline__ int shared_chunk(const Shared& p, int keys, int tile) {
    return max(1, ((keys + p.n_shared - 1) / p.n_shared + tile - 1) / tile) * tile;
}

// Block `block` of the shared sides.  False: there is no such part.
template <int ROWS, int TILE>
__device__ __forceinline__ bool family_item(const Shared& p, int block, int G, Item& it) {
    const int tiles = (p.most_members * G + ROWS - 1) / ROWS;
    const int split = block % p.n_shared, tile = block / p.n_shared % tiles, family = block / p.n_shared / tiles;
    it.first_member = p.family_start[family];
    const int count = min(min(p.family_start[family + 1], p.n_members) - it.first_member, p.most_members);
    if (it.first_member < 0 || count <= 0) return false;
    it.row0 = tile * ROWS;
    it.rows = min(ROWS, count * G - it.row0);
    if (it.rows <= 0) return false;
    const int first = p.members[it.first_member];
    if (first < 0 || first >= p.n_seqs) return false;
    it.table = p.block_table + (size_t)first * p.table_stride;
    it.seq = -1;
    it.part = split;
    const int keys = shared_keys(p, first), chunk = shared_chunk(p, keys, TILE);          // (never beyond the table)
    it.begin = min(keys, split * chunk);
    it.end = min(keys, it.begin + chunk);
    return it.begin < it.end;
}
// The first of a sequence's own keys (its shared pages are whole already, unless the caller erred), and how many parts they make.
__device__ __forceinline__ int own_begin(const Shared& p, int seq) { return max(0, p.shared_len[seq]) / p.page_size * p.page_size; }
__device__ __forceinline__ int own_end(const Shared& p, int seq) { return min(p.kv_len[seq], p.table_stride * p.page_size); }
__device__ __forceinline__ int own_parts(const Shared& p, int seq) {
    return min(p.n_own, max(0, own_end(p, seq) - own_begin(p, seq) + p.own_chunk - 1) / p.own_chunk);
}
// Block `block` of the sequences' own sides, the first parts of all sequences first.  False: the sequence has no such part.
template <int ROWS>
__device__ __forceinline__ bool own_item(const Shared& p, int block, int G, Item& it) {
    const int tiles = (G + ROWS - 1) / ROWS, split = block / (p.n_seqs * tiles);
    block -= split * p.n_seqs * tiles;
    it.seq = block / tiles;
    it.row0 = block % tiles * ROWS;
    it.rows = min(ROWS, G - it.row0);
    it.first_member = 0;
    it.table = p.block_table + (size_t)it.seq * p.table_stride;
    it.part = p.n_shared + split;
    const int end = own_end(p, it.seq);
    it.begin = own_begin(p, it.seq) + split * p.own_chunk;
    it.end = min(end, it.begin + p.own_chunk);
    return it.begin < end;
}

// Lets an SM that runs `kernel` have as much of its memory shared as can be, so that a block of another kernel finds room beside it (once per device).
template <typename... KArgs>
int share_most(DeviceLimit& done, void (*kernel)(KArgs...)) {
    return done.allow(1, [](int* dev) { return (int)cudaGetDevice(dev); }, [&](size_t) {
        return (int)cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    });
}

// Blocks of the shared sides.
inline long long family_blocks(const Shared& p, int G, int rows) { return (long long)p.n_families * ((p.most_members * G + rows - 1) / rows) * p.n_shared; }

inline long long own_blocks(const Shared& p, int G, int rows) { return (long long)p.n_seqs * ((G + rows - 1) / rows) * p.n_own; }

// The pools as rows of D dimensions, a box a page of 64 of them with 128-byte swizzle, and the word of waits that ran out.
struct Maps {
    CUtensorMap k, v;
    unsigned int* error;
};

// The shared sides on the fifth-generation tensor cores (attention_shared_tcgen05.cu): head size 128, pages of 8 to 64 keys.
constexpr int kTcgen05Rows = 128;
int launch_tcgen05(const void* q, const Maps& maps, float* partial, const Shared& p, cudaStream_t stream);

}  // namespace shared_attention
}  // namespace pb
