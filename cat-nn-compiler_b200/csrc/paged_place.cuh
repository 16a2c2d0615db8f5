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

// The sequence of a new token, for tokens met in ascending order. A
// sequence's new tokens are rows [cu[seq], cu[seq + 1]), its last positions (cu
// null: token t is sequence t's only one).
struct Token {
    int seq = -1, end = -1;  // the sequence, and the row behind its last new token; seq < 0: none
    int len = 0;
    PLACE_FN void move_to(const int32_t* lens, const int32_t* cu, int seqs, int t) {
        if (seq >= 0 && t < end) return;
        seq = -1;
        if (!cu) {
            if (t >= seqs) return;
            seq = t;
            end = t + 1;
        } else {
            if (seqs < 1 || t < cu[0] || t >= cu[seqs]) return;
            int lo = 0, hi = seqs;  // the last sequence whose first token is at or before t
            while (hi - lo > 1) {
                const int mid = lo + ((hi - lo) >> 1);
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            end = cu[lo + 1];
            if (end <= t) return;  // starts that do not ascend
            seq = lo;
        }
        len = lens[seq];
    }
    // Its position, or -1 when it has none: a row before the first or behind
    // the last sequence, or one whose sequence ends before position 0.
    PLACE_FN int position(int t) const {
        const i64 pos = (i64)len - ((i64)end - t);
        return seq < 0 || pos < 0 ? -1 : (int)pos;
    }
};
PLACE_FN int token_position(const int32_t* lens, const int32_t* cu, int seqs, int t, int& seq) {
    Token at;
    at.move_to(lens, cu, seqs, t);
    seq = at.seq;
    return at.position(t);
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
