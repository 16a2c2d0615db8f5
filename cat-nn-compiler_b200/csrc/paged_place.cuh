// Where things lie in a paged cache: plain index arithmetic without any CUDA
// type, so that a host compiler takes it too and its bounds are checked
// without a GPU.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define PLACE_FN __host__ __device__ __forceinline__
#else
#define PLACE_FN inline
#endif

namespace catnn {
namespace place {

typedef int64_t i64;

// Position of new token t, its last `cu[seq+1] - cu[seq]` ones being a
// sequence's new tokens (cu null: token t is sequence t's only one), and the
// sequence it belongs to. -1 when it belongs to none: a row before the first
// or behind the last sequence, or one whose sequence ends before position 0.
PLACE_FN int token_position(const int32_t* lens, const int32_t* cu, i64 seqs, i64 t, i64& seq) {
    i64 end = t + 1;
    seq = t;
    if (cu) {
        if (seqs < 1 || t < cu[0] || t >= cu[seqs]) return -1;
        i64 lo = 0, hi = seqs;  // the last sequence whose first token is at or before t
        while (hi - lo > 1) {
            const i64 mid = (lo + hi) >> 1;
            if (cu[mid] <= t) lo = mid;
            else hi = mid;
        }
        seq = lo;
        end = cu[lo + 1];
        if (end <= t) return -1;  // starts that do not ascend
    } else if (t >= seqs) {
        return -1;
    }
    const i64 pos = (i64)lens[seq] - (end - t);
    return pos < 0 ? -1 : (int)pos;
}

// Index of the first element of kv head 0 at a position: caches [pages, hkv,
// page, hd]; a head further is page·hd elements on. -1 when the table has no
// such entry or the pool no such page.
PLACE_FN i64 cache_index(const int32_t* table, i64 seq, int pos, int page, int max_pages, i64 pages, int hkv, int hd) {
    if (pos < 0) return -1;
    const int slot = pos / page;
    if (slot >= max_pages) return -1;
    const int id = table[seq * max_pages + slot];
    if (id < 0 || id >= pages) return -1;
    return ((i64)id * hkv * page + (pos - slot * page)) * hd;
}

}  // namespace place
}  // namespace catnn
