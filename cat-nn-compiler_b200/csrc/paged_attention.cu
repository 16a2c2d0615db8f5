// Attention of one new token of each sequence against a paged cache:
//   o = softmax(q·Kᵀ/√hd)·V over the sequence's last min(len, window)
//   positions, lse = log Σ exp of the scaled scores.
// Position j of sequence b lies in slot j % page of the pool's page
// table[b][j / page]; a page is [Hkv, page, hd], so that one head's keys of a
// page are one run of memory.
//
// K and V are read once, 4 flops a byte and query head of the group, so HBM
// bounds it, and what matters is that every SM streams all the time whatever
// the lengths are. The work is cut into tiles of 32 positions of one
// sequence's kv head; all tiles in a row are dealt out evenly to the warps of
// a grid that fills the SMs once. A warp is on its own: its ring of cp.async
// tiles runs on across the sequences, there is no block barrier, and a running
// maximum and sum carry the softmax. What a warp has of a (sequence, head)
// that it shares with others goes to the workspace, and a second, dependent
// kernel joins those in order; a (sequence, head) of one warp is written at once.
//
// Measured: 64 sequences up to 6000, 16 query and 4 kv heads of 128, bf16, 388
// MB of cache: 73 us (0.81 of the copy rate); one sequence of 2047, 16 heads
// of 64: 6.6 us; 49.5 K positions of 2 kv heads of 64, fp32, 51 MB: 22.0 us.
// A warp that comes from one sequence to the next passes those of no length one
// by one: four of 1000 among 64, 256 and 1024 take 13.9, 24 and 80 us.
#include <algorithm>
#include <climits>

#include "ops.cuh"
#include "paged_place.cuh"
#include "tc_prims.cuh"

namespace catnn {
namespace paged {

constexpr int MAX_HD = 128;
constexpr int TK = 32;         // positions of a tile: one a lane
constexpr int MAX_CHUNKS = 512;

struct Args {
    const void *q, *kc, *vc;
    void* o;
    float* lse;
    const int32_t *table, *lens;
    i64 seqs;
    int h, hkv, hd, page, max_pages, window;
    i64 pages, q_stride;
    float scale;
    int* err;
    // tiles: a sequence's segments are its kv heads times the tiles of `rows` query heads of a group
    int rows, row_tiles, workers, pitch;  // pitch: floats of a row in `part`
    float *part, *ml;                     // [workers][2][rows][pitch] sums, [workers][2][rows][2] maximum and weight
};

// The positions [first, len) that sequence b attends to: its window, as far as
// the table holds it (nothing, where the window lies beyond the table).
__device__ __forceinline__ void span_of(const Args& a, i64 b, int& first, int& len) {
    const i64 held = (i64)a.max_pages * a.page;  // (with 32 bits k_paged_fma is compiled to 25.3 us in place of 21.3 on the long case)
    const int all = max(a.lens[b], 0);
    len = (int)min(held, (i64)all);
    first = a.window > 0 && all > a.window ? min(all - a.window, len) : 0;
}
__device__ __forceinline__ int tiles_of(const Args& a, i64 b) {  // of one segment
    int first, len;
    span_of(a, b, first, len);
    return (len - first + TK - 1) / TK;
}

__device__ __forceinline__ int warp_sum_int(int v) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)v); }
__device__ __forceinline__ int warp_scan_int(int v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Tiles of all sequences (the host sees to it that they stay below 2^31) and
// how they are dealt out: `workers` warps take `each` tiles in a row, the
// first `more` one more. Up to 32 sequences a lane keeps its one's tiles;
// of more, shared memory the sums of chunks of them.
struct Count {
    int total, per, chunks, workers, each, more;
    int own;  // this lane's sequence's tiles, where there are no more than 32
    __device__ __forceinline__ int start(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int worker(int tile) const {  // the one that has it
        const int big = more * (each + 1);
        return tile < big ? tile / (each + 1) : more + (tile - big) / each;
    }
};
template <int W> __device__ __forceinline__ Count count_tiles(const Args& a, int* chunk) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, segs = a.hkv * a.row_tiles;
    Count c;
    if (a.seqs <= 32) {
        c.per = c.chunks = 0;
        c.own = lane < a.seqs ? tiles_of(a, lane) * segs : 0;
        c.total = warp_sum_int(c.own);
    } else {
        c.per = (int)max((i64)32, (a.seqs + MAX_CHUNKS - 1) / MAX_CHUNKS);
        c.chunks = (int)((a.seqs + c.per - 1) / c.per);
        for (int i = warp; i < c.chunks; i += W) {
            const i64 b1 = min(a.seqs, (i64)(i + 1) * c.per);
            int s = 0;
            for (i64 b = (i64)i * c.per + lane; b < b1; b += 32) s += tiles_of(a, b) * segs;
            s = warp_sum_int(s);
            if (lane == 0) chunk[i] = s;
        }
        __syncthreads();
        int s = 0;
        for (int i = lane; i < c.chunks; i += 32) s += chunk[i];
        c.own = 0;
        c.total = warp_sum_int(s);
    }
    c.workers = max(1, min(a.workers, c.total));
    c.each = c.total / c.workers;
    c.more = c.total - c.each * c.workers;
    return c;
}

// The tiles before sequence b, by a warp.
__device__ __forceinline__ int tiles_before(const Args& a, const Count& c, const int* chunk, i64 b) {
    const int lane = threadIdx.x & 31, segs = a.hkv * a.row_tiles;
    if (c.chunks == 0) return warp_sum_int(lane < b ? c.own : 0);
    const int in = (int)(b / c.per);
    int s = 0;
    for (int i = lane; i < in; i += 32) s += chunk[i];
    for (i64 x = (i64)in * c.per + lane; x < b; x += 32) s += tiles_of(a, x) * segs;
    return warp_sum_int(s);
}

// A place in the order of tiles: sequence, segment (kv head major, then row
// tile), tile of the segment.
struct At {
    i64 b;
    int seg, tile, tiles, first, len;
    __device__ __forceinline__ void enter(const Args& a) {
        span_of(a, b, first, len);
        tiles = (len - first + TK - 1) / TK;
    }
    __device__ __forceinline__ void next(const Args& a, int segs) {
        if (++tile < tiles) return;
        tile = 0;
        if (++seg < segs) return;
        seg = 0;
        do {
            tiles = 0;
            if (++b >= a.seqs) return;
            enter(a);
        } while (tiles == 0);
    }
};
// Where tile t is (0 <= t < total).
__device__ __forceinline__ At locate(const Args& a, const Count& c, const int* chunk, int t) {
    const int lane = threadIdx.x & 31, segs = a.hkv * a.row_tiles;
    At at;
    at.b = a.seqs;
    at.seg = at.tile = at.tiles = at.first = at.len = 0;
    // the first of 32 counts, one a lane, that reaches past t, which becomes the rest: its lane, or -1
    auto reach = [&](int n) {
        const int up = warp_scan_int(n, lane);
        const unsigned past = __ballot_sync(0xffffffffu, up > t);
        const int l = past ? __ffs(past) - 1 : 31;
        t -= __shfl_sync(0xffffffffu, past ? up - n : up, l);
        return past ? l : -1;
    };
    if (c.chunks == 0) {
        const int l = reach(c.own);
        if (l >= 0) at.b = l;
    } else {
        int i = 0, l = -1;
        for (; i < c.chunks && l < 0; i += l < 0 ? 32 : 0) {
            l = reach(i + lane < c.chunks ? chunk[i + lane] : 0);
            if (l >= 0) i += l;
        }
        const i64 b1 = min(a.seqs, (i64)(i + 1) * c.per);
        l = -1;
        for (i64 b0 = (i64)i * c.per; b0 < b1 && l < 0; b0 += 32) {
            l = reach(b0 + lane < b1 ? tiles_of(a, b0 + lane) * segs : 0);
            if (l >= 0) at.b = b0 + l;
        }
    }
    if (at.b >= a.seqs) return at;  // lengths that changed under the kernel: nothing to do, but no way astray
    at.enter(a);
    if (at.tiles == 0) return at;
    at.seg = t / at.tiles;
    at.tile = t - at.seg * at.tiles;
    return at;
}

// What a warp does with its tiles, whatever the type of the cache: a ring of
// S tiles of K and V rows, each row of hd values at a pitch of PITCH bytes
// (an odd number of 16-byte pieces: neither ldmatrix nor row-a-lane reads meet
// bank conflicts). Lane l looks up where row l of a tile lies, two
// tiles before it is fetched; rows without a position or a page are zeros and not in `mask`.
template <typename T, int HDP, int S> struct Ring {
    static constexpr int PITCH = HDP * (int)sizeof(T) + 16, VEC = 16 / (int)sizeof(T), PIECES = HDP / VEC;
    static constexpr int TILE = TK * PITCH, STAGE = 2 * TILE, BYTES = S * STAGE + 16 * ((S * 4 + 15) / 16);
    char* base;
    unsigned* mask;
    At at;         // the tile to look up next
    int look_left, left;  // tiles still to look up, to fetch
    // this lane's row of the next two tiles to fetch: kv head, slot of its page, page (-2: no position)
    int kvh[2], slot[2], id[2];

    __device__ __forceinline__ void look(const Args& a) {
        kvh[0] = kvh[1], slot[0] = slot[1], id[0] = id[1];
        id[1] = -2;
        if (look_left > 0) {
            const int pos = at.first + at.tile * TK + (threadIdx.x & 31);
            kvh[1] = at.seg / a.row_tiles;
            if (pos < at.len) {
                const int p = (unsigned)pos / (unsigned)a.page;
                slot[1] = pos - p * a.page;
                id[1] = a.table[at.b * a.max_pages + p];
            }
            --look_left;
            at.next(a, a.hkv * a.row_tiles);
            if (at.tiles == 0) look_left = 0;
        }
    }
    __device__ __forceinline__ void start(const Args& a, const At& first, int tiles) {
        at = first;
        look_left = left = tiles;
        kvh[1] = slot[1] = 0;
        look(a);
        look(a);
#pragma unroll
        for (int s = 0; s < S - 1; ++s) fetch(a, s);
    }
    __device__ __forceinline__ void fetch(const Args& a, int stage) {
        const int lane = threadIdx.x & 31;
        if (left > 0) {
            const bool on = id[0] >= 0 && id[0] < a.pages;
            if (a.err && !on && id[0] != -2) atomicExch(a.err, 1);
            const i64 off = on ? (((i64)id[0] * a.hkv + kvh[0]) * a.page + slot[0]) * a.hd : -1;
            const unsigned m = __ballot_sync(0xffffffffu, on);
            if (lane == 0) mask[stage] = m;
            const uint32_t to = tc::smem_u32(base + stage * STAGE);
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int idx = i * 32 + lane, row = idx / PIECES, c = idx - row * PIECES;
                const i64 o = __shfl_sync(0xffffffffu, off, row);
                const bool here = o >= 0 && c * VEC < a.hd;
                const i64 e = here ? o + c * VEC : 0;
                tc::cp_async16(to + row * PITCH + c * 16, (const T*)a.kc + e, here);
                tc::cp_async16(to + TILE + row * PITCH + c * 16, (const T*)a.vc + e, here);
            }
            --left;
            look(a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    template <int N> __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
        __syncwarp();
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Where a warp's sums of a segment go: to the result (out >= 0: the first
// head's row index), or to a slot of the workspace.
struct Dest {
    i64 out;    // b·h + first head, or -1
    i64 slot;   // row 0 of its slot in part / ml
    int rows;   // heads of this row tile
};
__device__ __forceinline__ Dest dest_of(const Args& a, const At& seg, int worker, bool first, bool whole) {
    const int group = a.h / a.hkv, kvh = seg.seg / a.row_tiles, r0 = (seg.seg - kvh * a.row_tiles) * a.rows;
    Dest d;
    d.rows = min(a.rows, group - r0);
    d.out = whole ? seg.b * a.h + kvh * group + r0 : -1;
    d.slot = ((i64)worker * 2 + (first ? 0 : 1)) * a.rows;
    return d;
}

// ------------------------------------------------------------ bf16: tensor cores
// The query heads of a group are the 16 rows of mma.m16n8k16 (R8 = 1: only 8
// of them in use), K the columns of the first product as it lies, P out of
// the scores' own registers, V by ldmatrix.trans. P is rounded to bf16 for the
// second product; its sum is of the unrounded weights.
template <int HDP, int R8, int S, int W>
__global__ void __launch_bounds__(W * 32) k_paged_mma(const __grid_constant__ Args a) {
    using R = Ring<bf16, HDP, S>;
    constexpr int KS = HDP / 16, NV = HDP / 8;
    extern __shared__ __align__(16) char raw[];
    __shared__ int chunk[MAX_CHUNKS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, segs = a.hkv * a.row_tiles;
    tc::launch_dependents();
    const Count c = count_tiles<W>(a, chunk);
    const int me = warp * gridDim.x + blockIdx.x;  // few warps: one an SM first
    if (me >= c.workers || c.total == 0) return;
    const int t0 = c.start(me), t1 = c.start(me + 1);
    R ring;
    ring.base = raw + warp * R::BYTES;
    ring.mask = (unsigned*)(ring.base + S * R::STAGE);
    At cur = locate(a, c, chunk, t0);
    if (cur.tiles == 0) return;
    ring.start(a, cur, t1 - t0);
    const float sc = a.scale * LOG2E;
    const uint32_t kaddr = (lane & 7) * R::PITCH + (lane >> 3) * 16;
    const uint32_t vaddr = ((lane & 7) + (lane >> 3 & 1) * 8) * R::PITCH + (lane >> 4) * 16;
    bool first = true;
    int stage = 0;
    for (int t = t0; t < t1 && cur.tiles > 0;) {
        // a segment, or this warp's part of it
        const int here = min(cur.tiles - cur.tile, t1 - t);
        const Dest d = dest_of(a, cur, me, first, here == cur.tiles);
        uint32_t qa[KS][R8 * 2];
        {
            const int group = a.h / a.hkv, kvh = cur.seg / a.row_tiles, r0 = (cur.seg - kvh * a.row_tiles) * a.rows;
            const bf16* q = (const bf16*)a.q + cur.b * a.q_stride + (i64)(kvh * group + r0) * a.hd;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int u = 0; u < R8 * 2; ++u) {
                    const int row = (lane >> 2) + (u % R8) * 8, col = k * 16 + (lane & 3) * 2 + (u / R8) * 8;
                    qa[k][u] = row < d.rows && col < a.hd ? *(const uint32_t*)(q + (i64)row * a.hd + col) : 0u;
                }
        }
        float m[R8], l[R8], o[NV][4];
#pragma unroll
        for (int r = 0; r < R8; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[n][u] = 0.f;
        for (int i = 0; i < here; ++i) {
            ring.template wait<S - 2>();
            ring.fetch(a, stage == 0 ? S - 1 : stage - 1);
            const uint32_t kb = tc::smem_u32(ring.base + stage * R::STAGE), vb = kb + R::TILE;
            const unsigned mask = ring.mask[stage];
            float s[TK / 8][4];
#pragma unroll
            for (int n = 0; n < TK / 8; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < KS; k += 2) {
                    uint32_t b[4];
                    tc::ldsm4(b, kb + n * 8 * R::PITCH + kaddr + k * 32);
                    const uint32_t a0[4] = {qa[k][0], R8 > 1 ? qa[k][1] : 0u, qa[k][R8], R8 > 1 ? qa[k][R8 * 2 - 1] : 0u};
                    const uint32_t a1[4] = {qa[k + 1][0], R8 > 1 ? qa[k + 1][1] : 0u, qa[k + 1][R8],
                                            R8 > 1 ? qa[k + 1][R8 * 2 - 1] : 0u};
                    tc::mma16816(s[n], a0, b[0], b[1]);
                    tc::mma16816(s[n], a1, b[2], b[3]);
                }
            }
            if (mask != 0xffffffffu) {
#pragma unroll
                for (int n = 0; n < TK / 8; ++n)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (!(mask >> (n * 8 + (lane & 3) * 2 + (u & 1)) & 1u)) s[n][u] = -INFINITY;
            }
            float keep[R8], mc[R8];
            bool moved = false;
#pragma unroll
            for (int r = 0; r < R8; ++r) {
                float top = m[r];
#pragma unroll
                for (int n = 0; n < TK / 8; ++n) top = fmaxf(top, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                mc[r] = top == -INFINITY ? 0.f : top * sc;
                keep[r] = ex2(m[r] * sc - mc[r]);
                moved |= top != m[r];
                m[r] = top;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int r = 0; r < R8; ++r) {
                        o[n][2 * r] *= keep[r];
                        o[n][2 * r + 1] *= keep[r];
                    }
#pragma unroll
                for (int r = 0; r < R8; ++r) l[r] *= keep[r];
            }
            uint32_t p[TK / 16][4];
#pragma unroll
            for (int n = 0; n < TK / 8; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t w = 0u;
                    if (r < R8) {
                        const float p0 = ex2(fmaf(s[n][2 * r], sc, -mc[r % R8])), p1 = ex2(fmaf(s[n][2 * r + 1], sc, -mc[r % R8]));
                        l[r % R8] += p0 + p1;
                        const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
                        w = *(const uint32_t*)&h;
                    }
                    p[n / 2][(n & 1) * 2 + r] = w;
                }
#pragma unroll
            for (int k = 0; k < TK / 16; ++k)
#pragma unroll
                for (int n = 0; n < NV; n += 2) {
                    uint32_t b[4];
                    tc::ldsm4_t(b, vb + k * 16 * R::PITCH + vaddr + n * 16);
                    tc::mma16816(o[n], p[k], b[0], b[1]);
                    tc::mma16816(o[n + 1], p[k], b[2], b[3]);
                }
            __syncwarp();
            if (++stage == S) stage = 0;
        }
#pragma unroll
        for (int r = 0; r < R8; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int row = (lane >> 2) + r * 8;
            if (row >= d.rows) continue;
            if (d.out >= 0) {
                const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
                bf16* to = (bf16*)a.o + (d.out + row) * a.hd + (lane & 3) * 2;
#pragma unroll
                for (int n = 0; n < NV; ++n)
                    if (n * 8 < a.hd)
                        *(__nv_bfloat162*)(to + n * 8) = l[r] == 0.f ? __floats2bfloat162_rn(0.f, 0.f)
                                                                     : __floats2bfloat162_rn(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
                if ((lane & 3) == 0) a.lse[d.out + row] = l[r] == 0.f ? -INFINITY : m[r] * a.scale + LN2 * log2f(l[r]);
            } else {
                float* to = a.part + (d.slot + row) * a.pitch + (lane & 3) * 2;
#pragma unroll
                for (int n = 0; n < NV; ++n)
                    if (n * 8 < a.hd) *(float2*)(to + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if ((lane & 3) == 0) *(float2*)(a.ml + (d.slot + row) * 2) = make_float2(m[r] * sc, l[r]);
            }
        }
        t += here;
        first = false;
        cur.tile = cur.tiles - 1;
        cur.next(a, segs);
    }
}

// ------------------------------------------------------------ fp32: FMA
// A lane has a position's scores for the first product and hd / 32 columns
// for the second; q and the weights pass through shared memory, from where
// whole warps read the same words. Shared memory's wavefronts bound it, so
// everything moves in the widest pieces there are.
template <int N> struct __align__(N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4) Floats {
    float v[N];
};
template <int HDP, int G, int S, int W>
__global__ void __launch_bounds__(W * 32) k_paged_fma(const __grid_constant__ Args a) {
    using R = Ring<float, HDP, S>;
    constexpr int C = HDP / 32;
    constexpr int WARP_BYTES = R::BYTES + G * (HDP + TK) * 4;
    extern __shared__ __align__(16) char raw[];
    __shared__ int chunk[MAX_CHUNKS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, segs = a.hkv * a.row_tiles;
    tc::launch_dependents();
    const Count c = count_tiles<W>(a, chunk);
    const int me = warp * gridDim.x + blockIdx.x;
    if (me >= c.workers || c.total == 0) return;
    const int t0 = c.start(me), t1 = c.start(me + 1);
    R ring;
    ring.base = raw + warp * WARP_BYTES;
    ring.mask = (unsigned*)(ring.base + S * R::STAGE);
    float* const qs = (float*)(ring.base + R::BYTES);  // [HDP / 4][G][4]
    float* const ps = qs + G * HDP;                    // [TK][G]
    At cur = locate(a, c, chunk, t0);
    if (cur.tiles == 0) return;
    ring.start(a, cur, t1 - t0);
    const float sc = a.scale * LOG2E;
    bool first = true;
    int stage = 0;
    for (int t = t0; t < t1 && cur.tiles > 0;) {
        const int here = min(cur.tiles - cur.tile, t1 - t);
        const Dest d = dest_of(a, cur, me, first, here == cur.tiles);
        {
            const int group = a.h / a.hkv, kvh = cur.seg / a.row_tiles, r0 = (cur.seg - kvh * a.row_tiles) * a.rows;
            const float* q = (const float*)a.q + cur.b * a.q_stride + (i64)(kvh * group + r0) * a.hd;
            for (int i = lane; i < G * HDP; i += 32) {
                const int g = i / HDP, e = i - g * HDP;
                qs[(e / 4 * G + g) * 4 + e % 4] = g < d.rows && e < a.hd ? q[(i64)g * a.hd + e] * sc : 0.f;
            }
            __syncwarp();
        }
        float m[G], l[G], o[G][C];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int u = 0; u < C; ++u) o[g][u] = 0.f;
        }
        for (int i = 0; i < here; ++i) {
            ring.template wait<S - 2>();
            ring.fetch(a, stage == 0 ? S - 1 : stage - 1);
            const char* kb = ring.base + stage * R::STAGE;
            const unsigned mask = ring.mask[stage];
            float s[G];
#pragma unroll
            for (int g = 0; g < G; ++g) s[g] = 0.f;
#pragma unroll 4
            for (int e = 0; e < HDP / 4; ++e) {
                const float4 k = *(const float4*)(kb + lane * R::PITCH + e * 16);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float4 q = *(const float4*)(qs + (e * G + g) * 4);
                    s[g] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[g]))));
                }
            }
            Floats<G> pw;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (!(mask >> lane & 1u)) s[g] = -INFINITY;
                const float top = fmaxf(m[g], warp_max(s[g])), mc = top == -INFINITY ? 0.f : top;
                const float keep = ex2(m[g] - mc), p = ex2(s[g] - mc);
                l[g] = l[g] * keep + p;
                if (top != m[g])
#pragma unroll
                    for (int u = 0; u < C; ++u) o[g][u] *= keep;
                m[g] = top;
                pw.v[g] = p;
            }
            *(Floats<G>*)(ps + lane * G) = pw;
            __syncwarp();
            const char* vb = kb + R::TILE + lane * C * 4;
#pragma unroll 4
            for (int j = 0; j < TK; ++j) {
                const Floats<C> v = *(const Floats<C>*)(vb + j * R::PITCH);
                const Floats<G> p = *(const Floats<G>*)(ps + j * G);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int u = 0; u < C; ++u) o[g][u] = fmaf(p.v[g], v.v[u], o[g][u]);
            }
            __syncwarp();
            if (++stage == S) stage = 0;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float sum = warp_sum(l[g]);
            if (g >= d.rows) continue;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int u = 0; u < C; ++u) {
                const int e = lane * C + u;
                if (e >= a.hd) continue;
                if (d.out >= 0) ((float*)a.o)[(d.out + g) * a.hd + e] = sum == 0.f ? 0.f : o[g][u] * inv;
                else a.part[(d.slot + g) * a.pitch + e] = o[g][u];
            }
            if (lane == 0) {
                if (d.out >= 0) a.lse[d.out + g] = sum == 0.f ? -INFINITY : LN2 * (m[g] + log2f(sum));
                else *(float2*)(a.ml + (d.slot + g) * 2) = make_float2(m[g], sum);
            }
        }
        t += here;
        first = false;
        cur.tile = cur.tiles - 1;
        cur.next(a, segs);
    }
}

// ------------------------------------------------------------ join
// A CTA to a (sequence, query head) and the next one a grid on: nothing to do
// where one warp had all of it; zeros and -inf where there is nothing to
// attend to; else the parts of the warps that shared it, each brought to the
// largest maximum. Threads take four columns, and several of them, by turns,
// the parts. Who shared what is found out while the first kernel still runs.
// Few heads can have many parts each: 256 threads to one then, 128 otherwise,
// so that the CTAs find their places while the first kernel still runs.
template <typename T, int JOIN>
__global__ void __launch_bounds__(JOIN, JOIN == 128 ? 10 : 3) k_paged_join(const __grid_constant__ Args a) {
    __shared__ int chunk[MAX_CHUNKS];
    const int segs = a.hkv * a.row_tiles, tid = threadIdx.x, group = a.h / a.hkv, quads = (a.hd + 3) / 4;
    __shared__ float4 sum[JOIN / 32][MAX_HD / 4];
    __shared__ float2 weight[JOIN / 32][MAX_HD / 4];
    const int lane = tid & 31, warp = tid >> 5;
    const int lq = quads <= 8 ? 8 : quads <= 16 ? 16 : 32;  // lanes that take a part's row together
    const int quad = lane & (lq - 1), turns = JOIN / lq, turn = tid / lq;
    const Count c = count_tiles<JOIN / 32>(a, chunk);
    bool waited = false;
    for (i64 out = blockIdx.x; out < a.seqs * a.h; out += gridDim.x) {
        const i64 b = out / a.h;
        const int head = (int)(out - b * a.h), kvh = head / group, rt = (head - kvh * group) / a.rows;
        const int row = head - kvh * group - rt * a.rows, tiles = tiles_of(a, b);
        if (a.err && tid == 0 && a.lens[b] > (i64)a.max_pages * a.page) atomicExch(a.err, 1);
        const int s = tiles_before(a, c, chunk, b) + (kvh * a.row_tiles + rt) * tiles;
        if (tiles == 0 || s + tiles > c.total) {  // nothing to attend to (or lengths that changed under the kernel)
            for (int i = tid; i < a.hd; i += JOIN) st((T*)a.o + out * a.hd + i, 0.f);
            if (tid == 0) a.lse[out] = -INFINITY;
            continue;
        }
        const int w0 = c.worker(s), w1 = c.worker(s + tiles - 1);
        if (w0 == w1) continue;
        const int parts = w1 - w0 + 1;
        // the first may have come here from another segment; the others start here
        const i64 slot0 = ((i64)w0 * 2 + (c.start(w0) < s ? 1 : 0)) * a.rows + row;
        if (!waited) {
            tc::grid_dependency_wait();
            waited = true;
        }
        float m = -INFINITY, w = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (quad < quads)
            for (int p0 = turn; p0 < parts; p0 += 4 * turns) {
                float2 ml[4];
                float4 u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = p0 + i * turns;
                    const i64 slot = p ? (i64)(w0 + p) * 2 * a.rows + row : slot0;
                    ml[i] = p < parts ? __ldcg((const float2*)(a.ml + slot * 2)) : make_float2(-INFINITY, 0.f);
                    u[i] = p < parts ? __ldcg((const float4*)(a.part + slot * a.pitch + quad * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x)), base = top == -INFINITY ? 0.f : top;
                float f = ex2(m - base);
                w *= f;
                v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
                m = top;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f = ex2(ml[i].x - base);
                    w = fmaf(f, ml[i].y, w);
                    v.x = fmaf(f, u[i].x, v.x);
                    v.y = fmaf(f, u[i].y, v.y);
                    v.z = fmaf(f, u[i].z, v.z);
                    v.w = fmaf(f, u[i].w, v.w);
                }
            }
        auto add = [&](float m2, float w2, float4 v2) {
            const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top, f = ex2(m - base), f2 = ex2(m2 - base);
            m = top;
            w = w * f + w2 * f2;
            v = make_float4(v.x * f + v2.x * f2, v.y * f + v2.y * f2, v.z * f + v2.z * f2, v.w * f + v2.w * f2);
        };
        for (int o = lq; o < 32; o <<= 1)
            add(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, w, o),
                make_float4(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o),
                            __shfl_xor_sync(0xffffffffu, v.z, o), __shfl_xor_sync(0xffffffffu, v.w, o)));
        if (warp > 0 && lane < quads) {
            sum[warp][lane] = v;
            weight[warp][lane] = make_float2(m, w);
        }
        __syncthreads();
        if (warp == 0 && lane < quads) {
            for (int u = 1; u < JOIN / 32; ++u) add(weight[u][lane].x, weight[u][lane].y, sum[u][lane]);
            const float inv = w == 0.f ? 0.f : 1.f / w;
            const float r[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (quad * 4 + u < a.hd) st((T*)a.o + out * a.hd + quad * 4 + u, w == 0.f ? 0.f : r[u]);
            if (quad == 0) a.lse[out] = w == 0.f ? -INFINITY : LN2 * (m + log2f(w));
        }
        __syncthreads();
    }
    if (!waited) tc::grid_dependency_wait();  // what comes after this kernel comes after the first one too
}

// ------------------------------------------------------------ any size and alignment
constexpr int WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) k_paged_any(const __grid_constant__ Args a) {
    __shared__ float sm[WARPS], sl[WARPS], so[WARPS][MAX_HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 b = blockIdx.x / a.h;
    const int head = (int)(blockIdx.x - b * a.h), kvh = head / (a.h / a.hkv);
    int first, len;
    span_of(a, b, first, len);
    if (a.err && threadIdx.x == 0 && a.lens[b] > len) atomicExch(a.err, 1);
    float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int d = lane + 32 * u;
        q[u] = d < a.hd ? ld((const T*)a.q + b * a.q_stride + (i64)head * a.hd + d) * a.scale : 0.f;
    }
    for (int j = first + warp; j < len; j += WARPS) {
        i64 row = place::cache_index(a.table, b, j, a.page, a.max_pages, a.pages, a.hkv, a.hd);
        if (row < 0) {
            if (a.err) atomicExch(a.err, 1);
            continue;
        }
        row += (i64)kvh * a.page * a.hd;
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = lane + 32 * u;
            if (d < a.hd) s = fmaf(q[u], ld((const T*)a.kc + row + d), s);
        }
        s = warp_sum(s);
        // a NaN score leaves the maximum and makes its weight NaN; while all are -inf their weights are 0
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float keep = expf(m - base), p = expf(s - base);
        l = l * keep + p;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = lane + 32 * u;
            if (d < a.hd) acc[u] = acc[u] * keep + p * ld((const T*)a.vc + row + d);
        }
        m = mn;
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) so[warp][lane + 32 * u] = acc[u];
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm[w]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total = fmaf(sl[w], expf(sm[w] - base), total);
    for (int d = threadIdx.x; d < a.hd; d += WARPS * 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v = fmaf(so[w][d], expf(sm[w] - base), v);
        st((T*)a.o + (b * a.h + head) * a.hd + d, total != 0.f ? v / total : 0.f);
    }
    if (threadIdx.x == 0) a.lse[b * a.h + head] = total != 0.f ? top + logf(total) : -INFINITY;
}

// ------------------------------------------------------------ launchers
// Warps and CTAs of the streaming kernels by type and head size: enough rings
// of two stages to keep the memory busy (a third stage, or as many warps more,
// made no call faster), and for fp32, whose warps have more to compute, as
// many as the SM's shared memory holds.
struct Fill {
    int warps, per_sm, rows;  // warps of a CTA, CTAs an SM, query heads of a row tile
};
static constexpr int mma_warps(int hd) { return hd <= 64 ? 4 : 5; }
static constexpr int fma_warps(int hd) { return hd <= 64 ? 6 : hd <= 96 ? 4 : 3; }
static Fill fill_of(int dtype, int hd, int group) {
    if (dtype == CATNN_BF16) return Fill{mma_warps(hd), hd <= 64 ? 2 : 1, group <= 8 ? 8 : 16};
    return Fill{fma_warps(hd), 1, group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8};
}
constexpr int STAGES = 2;

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Layout {
    size_t ml, bytes;
    int workers, rows, pitch;
};
static Layout layout(Context* c, i64 h, i64 hkv, i64 hd, int dtype) {
    const Fill f = fill_of(dtype, (int)hd, (int)(h / hkv));
    Layout l;
    l.workers = c->sm_count * f.per_sm * f.warps;
    l.rows = (int)std::min<i64>(f.rows, h / hkv);
    l.pitch = (int)((hd + 3) / 4 * 4);
    l.ml = align256((size_t)l.workers * 2 * l.rows * l.pitch * 4);
    l.bytes = l.ml + align256((size_t)l.workers * 2 * l.rows * 2 * 4);
    return l;
}

template <typename Kern> static void launch(Context* c, Kern k, int grid, int threads, size_t smem, const Args& a) {
    if (!c->raised.count((const void*)k)) {
        CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        c->raised.insert((const void*)k);
    }
    k<<<grid, threads, smem, c->stream>>>(a);
    launched(c);
}

template <int HDP, int R8> static void run_mma(Context* c, const Args& a, const Fill& f) {
    constexpr int W = mma_warps(HDP);
    launch(c, k_paged_mma<HDP, R8, STAGES, W>, c->sm_count * f.per_sm, W * 32, W * Ring<bf16, HDP, STAGES>::BYTES, a);
}
template <int HDP, int G> static void run_fma(Context* c, const Args& a, const Fill& f) {
    constexpr int W = fma_warps(HDP), BYTES = W * (Ring<float, HDP, STAGES>::BYTES + G * (HDP + TK) * 4);
    static_assert(BYTES + MAX_CHUNKS * 4 <= 232448, "shared memory of a CTA");
    launch(c, k_paged_fma<HDP, G, STAGES, W>, c->sm_count * f.per_sm, W * 32, BYTES, a);
}
template <int R8> static void run_mma_hd(Context* c, const Args& a, const Fill& f) {
    if (a.hd <= 32) run_mma<32, R8>(c, a, f);
    else if (a.hd <= 64) run_mma<64, R8>(c, a, f);
    else if (a.hd <= 96) run_mma<96, R8>(c, a, f);
    else run_mma<128, R8>(c, a, f);
}
template <int G> static void run_fma_hd(Context* c, const Args& a, const Fill& f) {
    if (a.hd <= 32) run_fma<32, G>(c, a, f);
    else if (a.hd <= 64) run_fma<64, G>(c, a, f);
    else if (a.hd <= 96) run_fma<96, G>(c, a, f);
    else run_fma<128, G>(c, a, f);
}

}  // namespace paged

using namespace paged;

size_t paged_attention_workspace(Context* c, i64, i64 h, i64 hkv, i64 hd, int dtype) {
    return layout(c, h, hkv, hd, dtype).bytes;
}

void paged_attention(Context* c, const void* q, i64 q_stride, const void* kc, const void* vc, const int32_t* table,
                     const int32_t* lens, void* o, float* lse, i64 seqs, i64 h, i64 hkv, i64 hd, i64 pages, i64 page,
                     i64 max_pages, i64 window, int dtype, void* work, int* err) {
    if (seqs == 0) return;
    const Layout l = layout(c, h, hkv, hd, dtype);
    Args a{q, kc, vc, o, lse, table, lens, seqs, (int)h, (int)hkv, (int)hd, (int)page, (int)max_pages, (int)window, pages,
           q_stride, 1.0f / sqrtf((float)hd), err, l.rows, cdiv(h / hkv, l.rows), l.workers, l.pitch, (float*)work,
           (float*)((char*)work + l.ml)};
    const int vec = dtype == CATNN_BF16 ? 8 : 4;
    if (hd % vec != 0 || !aligned_to(kc, 16) || !aligned_to(vc, 16) || !aligned_to(q, 4) || (seqs > 1 && q_stride % 2 != 0) ||
        !aligned_to(o, 4)) {
        if (dtype == CATNN_BF16) k_paged_any<bf16><<<(int)(seqs * h), WARPS * 32, 0, c->stream>>>(a);
        else k_paged_any<float><<<(int)(seqs * h), WARPS * 32, 0, c->stream>>>(a);
        launched(c);
        return;
    }
    const i64 most = max_pages * page, reach = window > 0 ? std::min(most, window) : most;
    CATNN_CHECK(seqs * hkv * a.row_tiles <= INT_MAX / (reach / TK + 2), CATNN_ERR_UNSUPPORTED,
                "paged_attention: the table's positions times the heads pass 2^31 tiles of 32");
    const Fill f = fill_of(dtype, (int)hd, (int)(h / hkv));
    if (dtype == CATNN_BF16) {
        if (f.rows == 8) run_mma_hd<1>(c, a, f);
        else run_mma_hd<2>(c, a, f);
    } else {
        if (f.rows == 1) run_fma_hd<1>(c, a, f);
        else if (f.rows == 2) run_fma_hd<2>(c, a, f);
        else if (f.rows == 4) run_fma_hd<4>(c, a, f);
        else run_fma_hd<8>(c, a, f);
    }
    const bool few = seqs * h <= 2 * c->sm_count;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<i64>(seqs * h, (i64)c->sm_count * 10));
    cfg.blockDim = dim3(few ? 256 : 128);
    cfg.stream = c->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (dtype == CATNN_BF16) CUDA_OK(cudaLaunchKernelEx(&cfg, few ? k_paged_join<bf16, 256> : k_paged_join<bf16, 128>, a));
    else CUDA_OK(cudaLaunchKernelEx(&cfg, few ? k_paged_join<float, 256> : k_paged_join<float, 128>, a));
    launched(c);
}

}  // namespace catnn
