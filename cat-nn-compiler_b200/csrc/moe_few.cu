// A whole mixture-of-experts layer for a few tokens (at most 64):
//   logits = x·gate; the k largest, ties to the lower index; w = softmax
//   over those k; y = Σ_j w_j·(silu(x·w1)·(x·w3))·w2 of the j-th expert.
// The grouped GEMMs of the block for many tokens pad every expert to 128
// rows and take nine launches; here two kernels read the chosen experts'
// weights once, the first forming h, the second y. HBM bounds them while they
// stream; with few tokens the routing before the stream, the hand-over of h
// and the last sum take as long again.
//
// Measured at hidden 1024, mid 3584, 8 experts, top 2: bf16 1 token 19.0 us
// (44 MB of weights, 2.3 TB/s), 8 tokens 33.9, 64 tokens 47.4 (176 MB, 3.7
// TB/s); the block for many tokens takes 267, 310 and 319. fp32 1 token 29.2
// (88 MB), 16 tokens 76, 64 tokens 168 (352 MB; the FMAs of 16 tokens an
// expert, and 448 tiles on 296 places). 7 tokens, hidden 256, mid 512, fp32:
// 12.7 us.
//
// That is for hidden and mid of 64 and more, multiples of 8 (fp32: 4), and
// operands on 16-byte boundaries. For the rest k_up_any and k_down_any keep the
// call whole, one thread to a column, with every token reading its experts'
// weights for itself: 1.2 to 1.8 ms at hidden 1022, mid 3582.
#include <cooperative_groups.h>

#include <algorithm>

#include "ops.cuh"
#include "tc_prims.cuh"

namespace cg = cooperative_groups;

namespace catnn {
namespace few {

constexpr int MAX_E = 32, MAX_T = CATNN_MOE_FEW_MAX_TOKENS;
constexpr int THREADS = 128, NW = THREADS / 32;

struct Args {
    const void *x, *gate, *w1, *w3, *w2;
    void* y;
    float* h;  // [T·k, mid]
    int T, hidden, mid, E, k;
};

// The k choices of one row of logits and their softmax, as the router of the
// large block makes them: the largest remaining logit, ties to the lower index.
__device__ __forceinline__ void choose(const float* logit, int E, int k, int* idx, float* w) {
    unsigned taken = 0u;
    float top = 0.f, sum = 0.f;
    for (int j = 0; j < k; ++j) {
        int best = -1;
        float bv = 0.f;
        for (int e = 0; e < E; ++e) {
            if (taken >> e & 1u) continue;
            if (best < 0 || logit[e] > bv) {
                best = e;
                bv = logit[e];
            }
        }
        taken |= 1u << best;
        if (j == 0) top = bv;
        idx[j] = best;
        w[j] = expf(bv - top);
        sum += w[j];
    }
    const float inv = 1.f / fmaxf(sum, 1e-30f);
    for (int j = 0; j < k; ++j) w[j] *= inv;
}

// Routes token t with the whole CTA.
template <typename T>
__device__ __forceinline__ void route(const Args& a, int t, float* logit, int* idx, float* w) {
    const T* x = (const T*)a.x + (i64)t * a.hidden;
    const T* g = (const T*)a.gate;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = warp; e < a.E; e += NW) {
        float s = 0.f;
        for (int i = lane; i < a.hidden; i += 32) s = fmaf(ld(x + i), ld(g + (i64)i * a.E + e), s);
        s = warp_sum(s);
        if (lane == 0) logit[e] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) choose(logit, a.E, a.k, idx, w);
    __syncthreads();
}

// h[t·k + j][col] for one column a thread.
template <typename T>
__global__ void __launch_bounds__(THREADS) k_up_any(const __grid_constant__ Args a) {
    __shared__ float logit[MAX_E], w[MAX_E];
    __shared__ int idx[MAX_E];
    const int t = blockIdx.y, col = blockIdx.x * THREADS + threadIdx.x;
    route<T>(a, t, logit, idx, w);
    if (col >= a.mid) return;
    const T* x = (const T*)a.x + (i64)t * a.hidden;
    for (int j = 0; j < a.k; ++j) {
        const i64 at = (i64)idx[j] * a.hidden * a.mid + col;
        float u = 0.f, v = 0.f;
        for (int i = 0; i < a.hidden; ++i) {
            const float xi = ld(x + i);
            u = fmaf(xi, ld((const T*)a.w1 + at + (i64)i * a.mid), u);
            v = fmaf(xi, ld((const T*)a.w3 + at + (i64)i * a.mid), v);
        }
        a.h[((i64)t * a.k + j) * a.mid + col] = u / (1.f + expf(-u)) * v;
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) k_down_any(const __grid_constant__ Args a) {
    __shared__ float logit[MAX_E], w[MAX_E];
    __shared__ int idx[MAX_E];
    const int t = blockIdx.y, col = blockIdx.x * THREADS + threadIdx.x;
    route<T>(a, t, logit, idx, w);
    if (col >= a.hidden) return;
    float y = 0.f;
    for (int j = 0; j < a.k; ++j) {
        const T* w2 = (const T*)a.w2 + (i64)idx[j] * a.mid * a.hidden + col;
        const float* h = a.h + ((i64)t * a.k + j) * a.mid;
        float s = 0.f;
        for (int i = 0; i < a.mid; ++i) s = fmaf(h[i], ld(w2 + (i64)i * a.hidden), s);
        y = fmaf(w[j], s, y);
    }
    st((T*)a.y + (i64)t * a.hidden + col, y);
}

// ------------------------------------------------------------ tensor cores
// bf16, hidden and mid multiples of 8. A CTA takes 16·CW columns of one chosen
// expert's matrix (w1 and w3 beside each other, or w2) and a run of its rows:
// TMA brings tiles of 64 rows into a ring, each of CW warps multiplies 16
// columns, and the expert's tokens are the N side of mma.m16n8k16, so that
// one token costs what eight do. The rows of x (or h) of just those tokens
// come by cp.async (bulk copies of 128 bytes a row cost the copy unit more
// than the weights did), at a pitch of 144 bytes so that ldmatrix meets no
// bank conflict. Weights are the M side, read by ldmatrix.trans out of the
// swizzled tiles. The runs of one tile lie in one cluster, which adds its
// parts up through distributed shared memory in rank order.
//
// Where few experts are chosen, they are found first, by every CTA of both
// kernels for itself (ALL = false): a slot of the grid is the slot-th of them.
// With more choices (nearly) every expert has some token: a slot is an
// expert, whose first tiles are fetched while the first kernel routes, and
// the second kernel, whose first tiles are fetched beside the first's last,
// reads what the first found (ALL = true).
//
// fp32 (multiples of 4) runs the same kernels with other hands: the tensor
// cores would round to TF32, so packed FMAs multiply, two k at a time. A lane
// has four columns (two of w1 and of w3, or four of w2) of up to 8 or 16
// tokens; the warps split a tile's rows, and more tokens between them. What
// bounds it beside HBM is the rows of x, 16 bytes that all lanes read at once
// cost the registers' port as much as 512: with one column to a lane 64 tokens
// took 264 us in place of 167 (hidden 1024, mid 3584). Its logits are TF32 products all the same, of both halves of every
// value without that of the two lower halves: a product is off by up to 7
// half-steps of fp32, which a sum of many of them hides and a single one does not.
constexpr int BK = 64;
template <typename T> constexpr int XPITCH = BK * (int)sizeof(T) + 16;
template <typename T> constexpr int PIECE = 16 / (int)sizeof(T);
constexpr int SMEM_MAX = 144 * 1024;  // the widest ring and what lies beside it

struct TcArgs {
    const void *x, *gate;
    void *h, *y;
    float* yp;        // [runs][T·k, hidden]: each pair's share of y from each run of rows, before its weight
    unsigned* taken;  // [T], then [T·k] weights: what the first kernel found (ALL)
    unsigned* count;  // [column tiles of hidden][T]: shares of a token that are there
    int* status;      // set to 1 when a wait ran out
    long long patience;  // cycles after which a wait gives up; 0: the copying warps give up before their first tile
    int T, hidden, mid, E, k;
    int up_run, down_run;  // rows of a matrix that one CTA takes
    int counts;
};

// What routing leaves in shared memory. Pair t·k + i of token t is its i-th
// chosen expert by index.
struct Routes {
    unsigned* taken;  // [T] a token's experts as bits
    float* w;         // [T·k]
    short* tok;       // [T] tokens of this CTA's expert
    short* pair;      // [T] their pairs
    int expert, n, active;
};

static size_t routes_bytes(int T, int k) { return (size_t)T * (4 + 4 * k + 4); }

// Routing. A CTA routes 16 tokens (all of them, when there are no more); of
// more tokens each CTA of a cluster routes its share and tells the others, so
// that x is not read whole by every CTA. Logits are fp32 sums of exact bf16
// products by mma.sync. A warp takes every CW-th run of 32 k: a lane loads 8
// consecutive k of a token (the fragment layout's lane takes its k in that
// order; a sum does not care) and one gate row, which ldmatrix.trans turns by
// way of shared memory in the same order. A batch's loads are all in flight
// before the first is used: memory latency is what routing costs, and both
// kernels pay it.
constexpr int RT = 16;

// A float as an unsigned number in the same order; -0 as 0.
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The k choices of one token by a warp, lane e holding expert e's logit: the
// largest remaining one, ties to the lower index. NaN is as in a scan that
// takes the first remaining expert and then any larger one: a NaN is taken
// when it comes first and never otherwise.
__device__ __forceinline__ unsigned choose(float l, int E, int k, int lane, float& top) {
    const unsigned all = E == 32 ? 0xffffffffu : (1u << E) - 1u;
    const bool nan = l != l;
    const unsigned key = order_key(l);
    unsigned taken = 0u;
    top = 0.f;
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
        const unsigned left = all & ~taken;
        unsigned mine = left >> lane & 1u ? (nan ? (left & (0u - left)) == 1u << lane ? 0xffffffffu : 1u : key) : 0u;
        const unsigned best = __reduce_max_sync(0xffffffffu, mine);
        const int e = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
        if (j == 0) top = __shfl_sync(0xffffffffu, l, e);
        taken |= 1u << e;
    }
    return taken;
}

// fp32 logits of token t by a warp, lane e holding expert e's: an infinite
// value, or one that TF32 rounds to infinity, leaves NaN as its lower half,
// so logits that came out NaN are added up again from the values as they are
// (an expert shut off by -inf then has the logit -inf). Not where the token's
// own row has a NaN or an infinity, as stale rows of a padded batch may: then
// every logit is infinite or NaN, and the weights are NaN whichever are chosen.
__device__ __forceinline__ float exact_where_nan(const TcArgs& a, int t, float l) {
    const int lane = threadIdx.x & 31;
    unsigned left = __ballot_sync(0xffffffffu, l != l);
    if (left == 0) return l;
    const float* x = (const float*)a.x + (i64)t * a.hidden;
    bool finite = true;
#pragma unroll 8
    for (int i = lane; i < a.hidden; i += 32) finite &= fabsf(x[i]) < INFINITY;
    if (!__all_sync(0xffffffffu, finite)) return l;
    for (; left; left &= left - 1) {
        const int e = __ffs(left) - 1;
        float s = 0.f;
#pragma unroll 8
        for (int i = lane; i < a.hidden; i += 32) s = fmaf(x[i], ((const float*)a.gate)[(i64)i * a.E + e], s);
        s = warp_sum(s);
        if (lane == e) l = s;
    }
    return l;
}

// `issued` is called by every warp when its first batch's loads are on their way.
template <int R8, int CW, typename Issued>
__device__ __forceinline__ void logits_f32(const TcArgs& a, int t0, int rows, float* part, Issued issued) {
    constexpr int NB = 4;  // runs of 16 k in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, kj = (lane & 3) * 4;
    const int nt = (a.E + 7) / 8, ep = nt * 8;
    const float* xrow[R8];
#pragma unroll
    for (int i = 0; i < R8; ++i) xrow[i] = (const float*)a.x + (i64)(t0 + min(i * 8 + row, rows - 1)) * a.hidden + kj;
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
        const float* gcol = (const float*)a.gate + (i64)kj * a.E + min(j * 8 + row, a.E - 1);
        float acc[4] = {}, low[4] = {};
#pragma unroll 1
        for (int k0 = warp * 16; k0 < a.hidden; k0 += NB * CW * 16) {
            float x[NB][R8][4], g[NB][4];
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int k1 = k0 + q * CW * 16;
                const bool on = k1 + kj < a.hidden;  // hidden is a multiple of 4
#pragma unroll
                for (int i = 0; i < R8; ++i) {
                    const float4 v = on ? *(const float4*)(xrow[i] + k1) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[q][i][0] = v.x, x[q][i][1] = v.y, x[q][i][2] = v.z, x[q][i][3] = v.w;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) g[q][u] = on ? gcol[(i64)(k1 + u) * a.E] : 0.f;
            }
            if (j == 0 && k0 == warp * 16) issued();
#pragma unroll
            for (int q = 0; q < NB; ++q)
#pragma unroll
                for (int v = 0; v < 4; v += 2) {  // the instruction's k and k + 4 are a lane's two neighbours
                    uint32_t ah[4] = {}, al[4] = {}, bh[2], bl[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int i = 0; i < R8; ++i) {
                            ah[u * 2 + i] = tc::to_tf32(x[q][i][v + u]);
                            al[u * 2 + i] = tc::to_tf32(x[q][i][v + u] - __uint_as_float(ah[u * 2 + i]));
                        }
                        bh[u] = tc::to_tf32(g[q][v + u]);
                        bl[u] = tc::to_tf32(g[q][v + u] - __uint_as_float(bh[u]));
                    }
                    tc::mma1688_tf32(acc, ah, bh[0], bh[1]);
                    tc::mma1688_tf32(low, ah, bl[0], bl[1]);
                    tc::mma1688_tf32(low, al, bh[0], bh[1]);
                }
        }
        float* p = part + (warp * RT + row) * ep + j * 8 + (lane & 3) * 2;
        *(float2*)p = make_float2(acc[0] + low[0], acc[1] + low[1]);
        if (R8 > 1) *(float2*)(p + 8 * ep) = make_float2(acc[2] + low[2], acc[3] + low[3]);
    }
}
template <int R8, int CW, typename Issued>
__device__ __forceinline__ void logits_bf16(const TcArgs& a, int t0, int rows, char* gs, float* part, Issued issued) {
    constexpr int NB = R8 == 1 ? 8 : 4;  // runs of 32 k in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, kj = (lane & 3) * 8;
    const int nt = (a.E + 7) / 8, ep = nt * 8;
    gs += warp * NB * 512;
    const uint32_t gaddr = tc::smem_u32(gs) + (8 * ((lane & 7) >> 1) + (lane & 1) + 2 * (lane >> 3)) * 16;
    const bf16* xrow[R8];
#pragma unroll
    for (int i = 0; i < R8; ++i) xrow[i] = (const bf16*)a.x + (i64)(t0 + min(i * 8 + row, rows - 1)) * a.hidden + kj;  // a row past the last is not used
    // (the code is kept short: a launch meets its instructions cold, and their fetching costs as much as the data's)
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
        float acc[2][4] = {};
#pragma unroll 1
        for (int k0 = warp * 32; k0 < a.hidden; k0 += NB * CW * 32) {
            uint4 x[NB][R8];
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                const int k1 = k0 + q * CW * 32;
#pragma unroll
                for (int i = 0; i < R8; ++i)
                    x[q][i] = k1 + kj < a.hidden ? *(const uint4*)(xrow[i] + k1) : make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
            const bf16* grow = (const bf16*)a.gate + (i64)(k0 + lane) * a.E + j * 8;
            if (a.E % 8 == 0) {
                uint4 g[NB];
#pragma unroll
                for (int q = 0; q < NB; ++q)
                    g[q] = k0 + q * CW * 32 + lane < a.hidden ? *(const uint4*)(grow + q * CW * 32 * a.E) : make_uint4(0, 0, 0, 0);
                if (j == 0 && k0 == warp * 32) issued();
#pragma unroll
                for (int q = 0; q < NB; ++q) *(uint4*)(gs + q * 512 + lane * 16) = g[q];
            } else {
                if (j == 0 && k0 == warp * 32) issued();
                unsigned short* to = (unsigned short*)(gs + lane * 16);
#pragma unroll 1
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        to[q * 256 + e] = k0 + q * CW * 32 + lane < a.hidden && j * 8 + e < a.E
                                              ? ((const unsigned short*)grow)[q * CW * 32 * a.E + e] : (unsigned short)0;
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < NB; ++q) {
                uint32_t b[4];
                tc::ldsm4_t(b, gaddr + q * 512);
                const uint4 x0 = x[q][0], x1 = R8 == 1 ? make_uint4(0, 0, 0, 0) : x[q][R8 - 1];
                const uint32_t a0[4] = {x0.x, x1.x, x0.y, x1.y}, a1[4] = {x0.z, x1.z, x0.w, x1.w};
                tc::mma16816(acc[0], a0, b[0], b[1]);
                tc::mma16816(acc[1], a1, b[2], b[3]);
            }
        }
        float* p = part + (warp * RT + row) * ep + j * 8 + (lane & 3) * 2;
        *(float2*)p = make_float2(acc[0][0] + acc[1][0], acc[0][1] + acc[1][1]);
        if (R8 > 1) *(float2*)(p + 8 * ep) = make_float2(acc[0][2] + acc[1][2], acc[0][3] + acc[1][3]);
    }
}

// The expert of a slot and its tokens in order, from `taken`; every warp finds them for itself.
template <bool ALL, int CW> __device__ __forceinline__ void find_expert(const TcArgs& a, int slot, Routes& r) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned m0 = lane < a.T ? r.taken[lane] : 0u, m1 = lane + 32 < a.T ? r.taken[lane + 32] : 0u;
    unsigned any = __reduce_or_sync(0xffffffffu, m0 | m1);
    r.active = __popc(any);
    r.n = 0;
    int e = slot;
    if (!ALL) {
        r.expert = -1;
        if (slot >= r.active) return;
        for (int i = 0; i < slot; ++i) any &= any - 1;
        e = __ffs(any) - 1;
    }
    const unsigned bit = 1u << e, b0 = __ballot_sync(0xffffffffu, m0 & bit), b1 = __ballot_sync(0xffffffffu, m1 & bit);
    const unsigned below = (1u << lane) - 1u;
    r.expert = e;
    r.n = __popc(b0) + __popc(b1);
    if (warp == CW) {  // the warp that copies their rows keeps the list
        if (m0 & bit) {
            const int at = __popc(b0 & below);
            r.tok[at] = (short)lane;
            r.pair[at] = (short)(lane * a.k + __popc(m0 & (bit - 1u)));
        }
        if (m1 & bit) {
            const int at = __popc(b0) + __popc(b1 & below);
            r.tok[at] = (short)(lane + 32);
            r.pair[at] = (short)((lane + 32) * a.k + __popc(m1 & (bit - 1u)));
        }
        __syncwarp();
    }
}

// Fills r.taken, and the weights: `w` in shared memory where it is not null, or
// with `tell`, `taken` and the weights in the workspace. `prefetch` is run by
// the copying warp as soon as the loads of x and the gate are under way (before
// them it would hold them up in the memory's queues).
template <typename T, int R8, int CW, typename Prefetch>
__device__ __forceinline__ void route_tc(const TcArgs& a, char* room, Routes& r, float* w_here, bool tell, Prefetch prefetch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cl = cg::this_cluster();
    const int shares = (a.T + RT - 1) / RT, mine = shares > 1 ? (int)cl.block_rank() : 0;
    const int t0 = mine * RT, rows = min(RT, a.T - t0), ep = (a.E + 7) / 8 * 8;  // rows below 1: none of its own
    // waited for below: a peer's memory may be written once it has started
    if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float* part = (float*)room;           // [CW][RT][ep], then the warps' gate rows
    const auto issued = [] { asm volatile("bar.arrive 1, %0;" ::"n"((CW + 1) * 32) : "memory"); };
    if (warp == CW) {
        asm volatile("bar.sync 1, %0;" ::"n"((CW + 1) * 32) : "memory");
        prefetch();
    } else if (rows > 0 && warp * (64 / (int)sizeof(T)) < a.hidden) {
        if constexpr (sizeof(T) == 4) logits_f32<R8, CW>(a, t0, rows, part, issued);
        else logits_bf16<R8, CW>(a, t0, rows, room + CW * RT * MAX_E * 4, part, issued);
    } else {
        issued();
        for (int i = lane; i < RT * ep; i += 32) part[warp * RT * ep + i] = 0.f;
    }
    if (shares > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    unsigned* to = r.taken;  // lane p's copy of it
    if (shares > 1) to = cl.map_shared_rank(r.taken, min(lane, (int)cl.num_blocks() - 1));
    const int copies = shares > 1 ? (int)cl.num_blocks() : 1;
#pragma unroll 1
    for (int i = warp; i < rows; i += CW + 1) {
        float l = 0.f, top;
        if (lane < a.E)
#pragma unroll
            for (int w = 0; w < CW; ++w) l += part[(w * RT + i) * ep + lane];
        const int t = t0 + i;
        if constexpr (sizeof(T) == 4) l = exact_where_nan(a, t, l);
        const unsigned taken = choose(l, a.E, a.k, lane, top);
        if (lane < copies) to[t] = taken;
        if (w_here || tell) {
            const bool in = taken >> lane & 1u;
            float w = in ? expf(l - top) : 0.f;
            w /= fmaxf(warp_sum(w), 1e-30f);
            const int at = t * a.k + __popc(taken & ((1u << lane) - 1u));
            if (in && w_here) w_here[at] = w;
            if (tell) {
                if (in) ((float*)(a.taken + a.T))[at] = w;
                if (lane == 0) a.taken[t] = taken;
            }
        }
    }
    tc::fence_proxy_async();  // `part` and the gate rows lie where TMA writes next
    if (shares > 1) cl.sync();
    else __syncthreads();
}

// One CTA's product: M matrices (2: w1 and w3; 1: w2), CW warps of 16 columns,
// up to 8·NT tokens, ROOM bytes for the ring. A stage takes the room of its
// weights and of as many token rows as the expert has, so that the usual few
// tokens leave room for more stages.
constexpr int MAX_STAGES = 8;
template <typename T, bool ALL, int M, int NT, int BN_, int CW, int ROOM> struct Tc {
    static constexpr int ES = sizeof(T), BN = BN_, BOX = BN < 128 / ES ? BN : 128 / ES, THREADS = (CW + 1) * 32;
    static constexpr int KG = CW * 16 / BN;    // bf16: groups of warps that have the same columns and split a tile's k
    static constexpr int G = NT < 4 ? 8 : 16;  // fp32: tokens of a warp at most
    static constexpr int COLS = M * BN / 32;   // fp32: columns of a lane, those of w1 before those of w3
    static_assert(ES == 2 || (BN % 32 == 0 && NT * 8 <= G * CW && BK / CW % 4 == 0), "fp32: whole lanes and steps of four rows");
    static constexpr int W_BYTES = M * BK * BN * ES, RED_PITCH = BN + 4;  // bytes; floats
    static constexpr int RED = (ES == 4 ? CW * M * G : KG * M * NT * 8) * RED_PITCH;  // floats of all sums
    static constexpr int MIN_STAGES = ROOM / (W_BYTES + NT * 8 * XPITCH<T>);
    static constexpr int PRE = ALL ? (MIN_STAGES < 3 ? MIN_STAGES : 3) : 0;  // stages filled before routing
    static constexpr int SCRATCH = CW * (RT * MAX_E * 4 + (ES == 4 ? 0 : (NT == 1 ? 8 : 4) * 512));
    static_assert(ROOM % 1024 == 0 && MIN_STAGES >= 2, "two stages at least");
    static_assert(RED * 4 <= ROOM && (M == 1 && ALL ? 0 : PRE * W_BYTES + SCRATCH) <= ROOM,
                  "the parts, and routing beside the first stages, lie in the ring");
    static constexpr int BESIDE = 1024 + 2 * MAX_STAGES * 8 + 16;  // the ring's alignment, barriers, `stop`
    static_assert(ROOM + BESIDE + MAX_T * (8 + 4 * MAX_E) <= SMEM_MAX, "smem()'s largest");
    static size_t smem(int tokens, int k) { return ROOM + BESIDE + routes_bytes(tokens, k); }

    // fp32: a tile's tokens are split over 2^teams(n) teams of warps, G or fewer to each
    static __device__ __forceinline__ int teams(int n) {
        return ES == 2 || NT * 8 <= G ? 0 : (n > G) + (n > 2 * G) + (n > 4 * G);
    }
    // groups of warps with the same columns and tokens, that split a tile's k; rows of a group's sums of one matrix
    static __device__ __forceinline__ int groups(int n) { return ES == 4 ? CW >> teams(n) : KG; }
    static __device__ __forceinline__ int red_rows(int n) { return ES == 4 ? G << teams(n) : NT * 8; }

    char* ring;
    uint64_t *full, *empty;
    int* stop;  // not 0: a wait of this CTA ran out
    const CUtensorMap* w[2];
    int r0, r1, col0, iters;

    __device__ __forceinline__ Tc(const TcArgs& a, char* raw, Routes& r, const CUtensorMap* w0, const CUtensorMap* w1, int run,
                                  int rows, int cols) {
        ring = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
        full = (uint64_t*)(ring + ROOM);
        empty = full + MAX_STAGES;
        stop = (int*)(empty + MAX_STAGES);
        r.taken = (unsigned*)(stop + 4);
        r.w = (float*)(r.taken + a.T);
        r.tok = (short*)(r.w + a.T * a.k);
        r.pair = r.tok + a.T;
        w[0] = w0;
        w[1] = w1;
        r0 = blockIdx.y * run;
        r1 = min(rows, r0 + run);
        col0 = blockIdx.x * BN;
        iters = r1 > r0 && col0 < cols ? (r1 - r0 + BK - 1) / BK : 0;
        if (threadIdx.x == CW * 32) {
            for (int s = 0; s < MAX_STAGES; ++s) {
                tc::mbar_init(&full[s], 1 + 32);  // the weights' bytes, and the copying warp's lanes
                tc::mbar_init(&empty[s], CW);
            }
            *stop = 0;
            tc::fence_mbar_init();
        }
    }
    // The slot's first tiles, by the copying warp.
    __device__ __forceinline__ void prefetch() const {
        if (threadIdx.x == CW * 32)
            for (int it = 0; it < PRE && it < iters; ++it) weights(it, it, blockIdx.z);
    }
    __device__ __forceinline__ void weights(int it, int st, int expert) const {
        char* at = ring + st * W_BYTES;
        tc::mbar_arrive_expect_tx(&full[st], W_BYTES);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < BN; c += BOX)
                tc::tma_load_3d(at + (m * BN + c) * BK * ES, w[m], col0 + c, r0 + it * BK, expert, &full[st]);
    }
    // A lane's wait for a phase; after one of the CTA's ran out the others have next to no patience left. The loops
    // go on all the same, with what is in the ring: a way out of them, which all lanes would have to agree on, cost 1.4
    // us at 64 tokens (bf16) and 8 in fp32.
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const TcArgs& a) const {
        if (tc::mbar_try_wait(tc::smem_u32(bar), parity)) return true;
        return tc::mbar_wait(bar, parity, stop, 1, *(volatile int*)stop ? 0 : a.patience, false);
    }
    // After a wait ran out, by the copying warp: let the last of the tiles that it asked for land in each of the stages
    // (whose sums come to lie there), which is a matter of microseconds, and leave word.
    __device__ __forceinline__ void settle(const TcArgs& a, int asked, int stages) const {
        for (int st = 0; st < stages && st < asked; ++st)
            if (!tc::mbar_wait(&full[st], (asked - 1 - st) / stages & 1, stop, 1, 4000000000ll, false)) break;
        atomicExch(a.status, 1);
    }
    // An expert that no token takes: let what was fetched land, then leave.
    __device__ __forceinline__ void drain(const TcArgs& a) const {
        if (threadIdx.x >= CW * 32)
            for (int it = 0; it < PRE && it < iters; ++it) {
                tc::mbar_arrive(&full[it]);
                tc::mbar_wait(&full[it], 0, a.status, 1, 4000000000ll, false);
            }
    }
};

// Rows [r0, r1) of the expert's matrices times the same columns of `rows`
// (row index `idx`, row length `len`), left in shared memory: sum(m, token
// index, column in the tile).
template <typename T, bool ALL, int M, int NT, int BN, int CW, int ROOM, typename Wait>
__device__ __forceinline__ void product(const Tc<T, ALL, M, NT, BN, CW, ROOM>& s, const TcArgs& a, const Routes& r, const short* idx,
                                        const T* rows, int len, Wait wait) {
    using S = Tc<T, ALL, M, NT, BN, CW, ROOM>;
    using namespace tc::pairs;
    constexpr bool F32 = sizeof(T) == 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int iters = s.iters, nte = (r.n + 7) / 8, xbytes = nte * 8 * XPITCH<T>;
    const int stages = min(MAX_STAGES, ROOM / (S::W_BYTES + xbytes));
    char* const xring = s.ring + stages * S::W_BYTES;
    float acc[F32 ? 1 : M][NT][4];  // bf16: the fragments
    constexpr int COLS = F32 ? S::COLS : 1;
    f2 sum[F32 ? S::G : 1][COLS];   // fp32: a token's even and odd k
#pragma unroll
    for (int m = 0; m < (F32 ? 1 : M); ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[m][j][u] = 0.f;
#pragma unroll
    for (int t = 0; t < (F32 ? S::G : 1); ++t)
#pragma unroll
        for (int c = 0; c < COLS; ++c) sum[t][c] = pack2(0.f, 0.f);
    // fp32: this warp's tokens [t0, t0 + G), of which `per` are its own, and its share of a tile's rows
    const int teams = S::teams(r.n), kg32 = warp >> teams;
    const int per = (((r.n + (1 << teams) - 1) >> teams) + 3) & ~3, t0 = (warp & (1 << teams) - 1) * per;
    int asked = 0;  // tiles that the copying warp asked for
    if (warp == CW) {
        auto tokens = [&](int it, int st) {
            constexpr int P = BK / PIECE<T>;  // 16-byte pieces of a row
            const uint32_t at = tc::smem_u32(xring + st * xbytes);
            const int k0 = s.r0 + it * BK, pieces = (min(s.r1, k0 + BK) - k0) / PIECE<T>;
            for (int i = lane; i < r.n * P; i += 32) {
                const int row = i / P, c = i % P;
                const bool on = c < pieces;
                tc::cp_async16(at + row * XPITCH<T> + c * 16, rows + (i64)idx[row] * len + (on ? k0 + c * PIECE<T> : 0), on);
            }
            tc::cp_async_arrive(&s.full[st]);
            ++asked;
        };
        bool lost = a.patience == 0;  // a wait of this lane's ran out: it asks for nothing more
        // weights first: they wait for nobody
        if (lane == 0 && !lost)
            for (int it = S::PRE; it < iters && it < stages; ++it) s.weights(it, it, r.expert);
        __syncwarp();
        wait();
        for (int it = 0; it < iters && it < (lost ? S::PRE : stages); ++it) tokens(it, it);
        for (int it = stages, st = 0, ph = 0; it < iters; ++it) {
            lost = lost || !s.wait(&s.empty[st], ph, a);
            if (lane == 0 && !lost) s.weights(it, st, r.expert);
            __syncwarp();
            if (!lost) tokens(it, st);
            if (++st == stages) st = 0, ph ^= 1;
        }
    } else if constexpr (F32) {
        wait();
        const int share = BK / CW << teams, mine = min(per, r.n - t0);
        for (int it = 0, st = 0, ph = 0; it < iters; ++it) {
            const int kk = min(BK, s.r1 - s.r0 - it * BK), k1 = min(kk, (kg32 + 1) * share);  // kk is a multiple of 4
            s.wait(&s.full[st], ph, a);
            const float* wt = (const float*)(s.ring + st * S::W_BYTES) + lane;
            const char* xt = xring + st * xbytes + t0 * XPITCH<T>;
#pragma unroll 1
            for (int k = kg32 * share; k < k1; k += 4) {
                f2 w[COLS][2];
#pragma unroll
                for (int c = 0; c < COLS; ++c) {  // boxes of 32 columns
                    const float* wc = wt + (c * BK + k) * 32;
                    w[c][0] = pack2(wc[0], wc[32]);
                    w[c][1] = pack2(wc[64], wc[96]);
                }
#pragma unroll
                for (int t = 0; t < S::G; t += 2) {
                    if (t >= mine) break;
                    ulonglong2 x[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) x[u] = *(const ulonglong2*)(xt + (t + u) * XPITCH<T> + k * 4);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int c = 0; c < COLS; ++c) {
                            sum[t + u][c] = fma2(w[c][0], x[u].x, sum[t + u][c]);
                            sum[t + u][c] = fma2(w[c][1], x[u].y, sum[t + u][c]);
                        }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.empty[st]);
            if (++st == stages) st = 0, ph ^= 1;
        }
    } else {
        wait();
        const int k8 = lane & 7, hi = lane >> 4 & 1, mid8 = lane >> 3 & 1;
        const int wm = warp % (BN / 16), kg = warp / (BN / 16);
        const uint32_t wcol = wm / (S::BOX / 16) * (BK * S::BOX * 2), chunk = wm % (S::BOX / 16) * 2 + mid8;
        for (int it = 0, st = 0, ph = 0; it < iters; ++it) {
            const int kk = min(BK, s.r1 - s.r0 - it * BK);
            s.wait(&s.full[st], ph, a);
            const uint32_t wb = tc::smem_u32(s.ring + st * S::W_BYTES) + wcol, xb = tc::smem_u32(xring + st * xbytes);
#pragma unroll
            for (int k2 = 0; k2 < BK; k2 += 32 * S::KG) {
                const int k0 = k2 + kg * 32;
                if (k0 >= kk) break;
                uint32_t wa[M][2][4];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    // 8x8 blocks of (k, column): (0, 0), (0, 8), (8, 0), (8, 8)
                    const int k = k0 + q * 16 + hi * 8 + k8;
#pragma unroll
                    for (int m = 0; m < M; ++m)
                        tc::ldsm4_t(wa[m][q], wb + m * BK * BN * 2 + k * S::BOX * 2 +
                                                  ((chunk ^ (S::BOX == 64 ? k & 7 : k >> 1 & 3)) << 4));
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (j >= nte) break;
                    uint32_t b[4];
                    tc::ldsm4(b, xb + (j * 8 + k8) * XPITCH<T> + (k0 / 8 + (lane >> 3)) * 16);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        tc::mma16816(acc[m][j], wa[m][0], b[0], b[1]);
                        tc::mma16816(acc[m][j], wa[m][1], b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.empty[st]);
            if (++st == stages) st = 0, ph ^= 1;
        }
    }
    __syncthreads();  // every tile of the ring has landed and been read, or a wait ran out
    const bool stopped = *(volatile int*)s.stop != 0;  // then the sums are NaN
    if (stopped) {
        if (warp == CW) s.settle(a, asked, stages);
        __syncthreads();
    }
    if (warp == CW) return;
    const float nan = __uint_as_float(0x7fc00000u);
    if constexpr (F32) {
        const int rows = S::red_rows(r.n);
#pragma unroll
        for (int t = 0; t < S::G; ++t)
            if (t < per && t0 + t < r.n)
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    ((float*)s.ring)[((kg32 * M + c / (BN / 32)) * rows + t0 + t) * S::RED_PITCH + c % (BN / 32) * 32 + lane] =
                        stopped ? nan : sum2(sum[t][c]);
    } else {
        const int wm = warp % (BN / 16), kg = warp / (BN / 16);
        float* red = (float*)s.ring + kg * M * NT * 8 * S::RED_PITCH + wm * 16 + (lane >> 2) + (lane & 3) * 2 * S::RED_PITCH;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (j >= nte) break;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    red[(m * NT * 8 + j * 8 + (u & 1)) * S::RED_PITCH + (u >> 1) * 8] = stopped ? nan : acc[m][j][u];
            }
    }
}

// Adds to v[m] four columns of token t of one CTA's sums of n tokens.
template <typename S, int M> __device__ __forceinline__ void add_sums(const float* red, int n, int t, int c, float4 (&v)[M]) {
    const int groups = S::groups(n), rows = S::red_rows(n);
#pragma unroll 4
    for (int g = 0; g < groups; ++g)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const float4 w = *(const float4*)(red + ((g * M + m) * rows + t) * S::RED_PITCH + c);
            v[m].x += w.x;
            v[m].y += w.y;
            v[m].z += w.z;
            v[m].w += w.w;
        }
}

template <typename T, bool ALL, int NT, int BN, int CW, int ROOM, int PER_SM>
__global__ void __launch_bounds__((CW + 1) * 32, PER_SM)
    k_up_tc(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap w1, const __grid_constant__ CUtensorMap w3) {
    extern __shared__ char raw[];
    tc::launch_dependents();  // the second kernel may take the SMs' free places and fetch w2
    Routes r;
    using S = Tc<T, ALL, 2, NT, BN, CW, ROOM>;
    const S s(a, raw, r, &w1, &w3, a.up_run, a.hidden, a.mid);
    if (blockIdx.y == 0 && blockIdx.z == 0)
        for (int i = blockIdx.x * S::THREADS + threadIdx.x; i < a.counts; i += gridDim.x * S::THREADS) a.count[i] = 0u;
    route_tc<T, NT == 1 ? 1 : 2, CW>(a, s.ring + S::PRE * S::W_BYTES, r, nullptr,
                                  ALL && blockIdx.x < cg::this_cluster().dim_blocks().x && blockIdx.z == 0, [&] { s.prefetch(); });
    find_expert<ALL, CW>(a, blockIdx.z, r);
    if (r.n == 0) {  // the whole cluster: it shares its slot
        s.drain(a);
        return;
    }
    __syncthreads();
    product(s, a, r, r.tok, (const T*)a.x, a.hidden, [] {});
    // the runs of a tile add their sums up in rank order, each a share of the tile
    cg::cluster_group cl = cg::this_cluster();
    const int runs = gridDim.y, run = blockIdx.y, cx = (int)cl.dim_blocks().x, ix = (int)cl.block_index().x;
    if (runs > 1) cl.sync();
    else __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x * runs + run; i < r.n * (BN / 4); i += S::THREADS * runs) {
        const int t = i / (BN / 4), c = (i - t * (BN / 4)) * 4;
        if (s.col0 + c >= a.mid) continue;
        float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int p = 0; p < runs; ++p)
            add_sums<S, 2>(runs > 1 ? cl.map_shared_rank((float*)s.ring, p * cx + ix) : (float*)s.ring, r.n, t, c, v);
        const float* u = (const float*)&v[0];
        const float* g = (const float*)&v[1];
        float h[4];
        // held in the type that the second product multiplies in (bf16 rounds it by up to 2^-8, and takes __expf)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = u[j] / (1.f + (sizeof(T) == 4 ? expf(-u[j]) : __expf(-u[j]))) * g[j];
        stv<T, 4>((T*)a.h + (i64)r.pair[t] * a.mid + s.col0 + c, h);
    }
    if (runs > 1) cl.sync();  // no CTA leaves while another reads its sums
}

template <typename T, bool ALL, int NT, int BN, int CW, int ROOM, int PER_SM>
__global__ void __launch_bounds__((CW + 1) * 32, PER_SM)
    k_down_tc(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap w2) {
    extern __shared__ char raw[];
    __shared__ bool last[MAX_T];
    Routes r;
    using S = Tc<T, ALL, 1, NT, BN, CW, ROOM>;
    const S s(a, raw, r, &w2, &w2, a.down_run, a.mid, a.hidden);
    if (ALL) {
        s.prefetch();
        tc::grid_dependency_wait();
        for (int i = threadIdx.x; i < a.T * (a.k + 1); i += S::THREADS) r.taken[i] = __ldcg(a.taken + i);
        __syncthreads();
    } else {
        route_tc<T, NT == 1 ? 1 : 2, CW>(a, s.ring, r, r.w, false, [] {});
    }
    find_expert<ALL, CW>(a, blockIdx.z, r);
    if (r.n == 0) {
        s.drain(a);
        return;
    }
    __syncthreads();
    const int col0 = s.col0;
    product(s, a, r, r.pair, (const T*)a.h, a.mid, [] { if (!ALL) tc::grid_dependency_wait(); });
    __syncthreads();
    const i64 run_size = (i64)a.T * a.k * a.hidden;
#pragma unroll 1
    for (int i = threadIdx.x; i < r.n * (BN / 4); i += S::THREADS) {
        const int t = i / (BN / 4), c = (i - t * (BN / 4)) * 4;
        if (col0 + c >= a.hidden) continue;
        float4 v[1] = {make_float4(0.f, 0.f, 0.f, 0.f)};
        add_sums<S, 1>((float*)s.ring, r.n, t, c, v);
        *(float4*)(a.yp + blockIdx.y * run_size + (i64)r.pair[t] * a.hidden + col0 + c) = v[0];
    }
    // Whoever brings the last share of a token's columns adds them up, expert
    // by expert and run by run, all loads on their way before the first is added.
    __threadfence();
    __syncthreads();
    for (int i = threadIdx.x; i < r.n; i += S::THREADS)
        last[i] = atomicAdd(a.count + blockIdx.x * a.T + r.pair[i] / a.k, 1u) == (unsigned)a.k * gridDim.y - 1u;
    __syncthreads();
    __threadfence();
    constexpr int Q = BN / 4, TEAMS = S::THREADS / Q, FLIGHT = 8;
    const int c = col0 + threadIdx.x % Q * 4, team = threadIdx.x / Q, runs = gridDim.y;
    if (c >= a.hidden || team >= TEAMS) return;
#pragma unroll 1
    for (int i = team; i < r.n; i += TEAMS) {
        if (!last[i]) continue;
        const int t = r.pair[i] / a.k;
        const float* p = a.yp + (i64)t * a.k * a.hidden + c;
        int lj = 0, lq = 0, j = 0, q = 0;  // of the next share to load, to add
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), y = v;
#pragma unroll 1
        for (int left = a.k * runs; left > 0; left -= FLIGHT) {
            float4 u[FLIGHT];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                if (f >= left) break;
                u[f] = __ldcg((const float4*)(p + lq * run_size + (i64)lj * a.hidden));
                if (++lq == runs) lq = 0, ++lj;
            }
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                if (f >= left) break;
                v.x += u[f].x;
                v.y += u[f].y;
                v.z += u[f].z;
                v.w += u[f].w;
                if (++q == runs) {
                    const float w = r.w[t * a.k + j];
                    y.x = fmaf(w, v.x, y.x);
                    y.y = fmaf(w, v.y, y.y);
                    y.z = fmaf(w, v.z, y.z);
                    y.w = fmaf(w, v.w, y.w);
                    v = make_float4(0.f, 0.f, 0.f, 0.f);
                    q = 0;
                    ++j;
                }
            }
        }
        const float o[4] = {y.x, y.y, y.z, y.w};
        stv<T, 4>((T*)a.y + (i64)t * a.hidden + c, o);
    }
}

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// How many runs a matrix's rows are cut into (at most 8, a cluster): as many
// as the SMs hold CTAs at once, of at least two tiles each, so that all are
// resident. Runs are whole tiles of 64 rows, so the last ones may be shorter,
// or have none (1152 rows in 8 runs: six of 192); what such a CTA adds is zero.
static int runs_of(Context* c, i64 tiles, i64 rows, int per_sm) {
    int s = 1;
    while (s < 8 && tiles * 2 * s <= (i64)c->sm_count * per_sm && rows / (2 * s) >= 2 * BK) s *= 2;
    return s;
}

template <typename Kern, typename... A>
static void launch(Context* c, Kern k, int threads, dim3 grid, dim3 cluster, size_t smem, bool dependent, const A&... args) {
    if (!c->raised.count((const void*)k)) {
        CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
        // all of the SM's memory as shared: the second kernel's CTAs come to SMs that the first still holds
        CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        c->raised.insert((const void*)k);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = c->stream;
    cudaLaunchAttribute at[1];
    if (dependent) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
    } else {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {cluster.x, cluster.y, 1};
    }
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CUDA_OK(cudaLaunchKernelEx(&cfg, k, args...));
    launched(c);
}

// The grid of one product: column tiles x runs x experts. The first kernel's
// are in clusters that hold a tile's runs and as many CTAs as share the routing.
struct Plan {
    dim3 grid, cluster;
    int run;
};
static Plan plan(Context* c, int slots, int T, bool first, int rows, int cols, int bn, int per_sm) {
    const int tiles = cdiv(cols, bn), runs = runs_of(c, (i64)tiles * slots, rows, per_sm);
    int shares = 1;
    while (first && shares * RT < T) shares *= 2;
    const int cx = std::max(1, shares / runs);
    return {dim3(cdiv(tiles, cx) * cx, runs, slots), dim3(cx, runs), cdiv(cdiv(rows, runs), BK) * BK};
}

constexpr int K = 1024;
// Kernel shapes by the number of tokens: columns of a CTA, its warps, its ring, CTAs an SM.
template <bool ALL_, int NT_, int BU_, int CU_, int RU_, int PU_, int BD_, int CD_, int RD_, int PD_> struct Shape {
    static constexpr bool ALL = ALL_;
    static constexpr int NT = NT_, BU = BU_, CU = CU_, RU = RU_, PU = PU_, BD = BD_, CD = CD_, RD = RD_, PD = PD_;
};

// Whether a slot of the grid is an expert, or the chosen experts are found
// before anything is fetched. With few choices most experts' tiles would be
// fetched in vain. Hidden 1024, mid 3584, 8 experts, top 2: at 4 tokens 31.4 us
// found first against 29.8, at 16 tokens 41.4 against 36.4; 8 tokens' top 4 of 32
// (hidden 512, mid 1000) 38.7 against 26.2. fp32, whose matrices are twice as
// long: 4 tokens 55.3 us found first against 57.4, 16 tokens 89.4 against 82.9.
template <typename T> static bool slot_is_expert(i64 tokens, i64 E, i64 k) {
    return sizeof(T) == 4 ? tokens > 8 : tokens > 8 || tokens * k >= E;
}

// f(Shape) for a problem.
template <typename T, typename F> static void with_shape(Context* c, i64 tokens, i64 hidden, i64 mid, i64 E, i64 k, F f) {
    const bool all = slot_is_expert<T>(tokens, E, k);
    if constexpr (sizeof(T) == 4) {
        // short columns: narrow tiles for more CTAs (7 tokens, hidden 256: 12.6 against 12.9 us; 1 token, hidden 1024:
        // 30.6 against 28.9). Many tokens: eight warps in one CTA an SM where all tiles fit on the SMs at once, else
        // two CTAs of four (64 tokens, 8 experts: hidden 512, mid 1024 39.1 against 46.2 us; 1024, 3584 189 against 167).
        const bool small = hidden <= 256, once = (i64)cdiv(mid, 64) * E <= c->sm_count;
        if (tokens <= 8 && small) f(Shape<false, 1, 32, 4, 52 * K, 3, 64, 4, 52 * K, 3>());
        else if (tokens <= 8) f(Shape<false, 1, 64, 4, 72 * K, 3, 128, 4, 72 * K, 3>());
        else if (tokens <= 16 && small) f(Shape<true, 2, 32, 4, 52 * K, 3, 64, 4, 52 * K, 3>());
        else if (tokens <= 16) f(Shape<true, 2, 64, 8, 104 * K, 2, 128, 8, 104 * K, 2>());
        else if (tokens <= 32 && once) f(Shape<true, 4, 64, 8, 120 * K, 1, 128, 8, 120 * K, 1>());
        else if (tokens <= 32) f(Shape<true, 4, 64, 4, 104 * K, 2, 128, 4, 104 * K, 2>());
        else if (once) f(Shape<true, 8, 64, 8, 120 * K, 1, 128, 8, 120 * K, 1>());
        else f(Shape<true, 8, 64, 4, 104 * K, 2, 128, 4, 104 * K, 2>());
    } else {
        // the second product's tiles are as wide as the first's where narrow ones would not fit on the SMs at once
        // (40 tokens, hidden 2048, mid 704, 16 experts: 41.9 against 38.7 us)
        const bool wide = (i64)cdiv(hidden, 64) * E > (i64)c->sm_count * 2;
        if (!all) f(Shape<false, 1, 64, 4, 52 * K, 2, 64, 4, 52 * K, 3>());
        else if (tokens <= 32 && wide) f(Shape<true, 4, 128, 8, 104 * K, 2, 128, 8, 104 * K, 2>());
        else if (tokens <= 32) f(Shape<true, 4, 128, 8, 104 * K, 2, 64, 4, 104 * K, 2>());
        else if (wide) f(Shape<true, 8, 128, 8, 104 * K, 2, 128, 8, 104 * K, 2>());
        else f(Shape<true, 8, 128, 8, 104 * K, 2, 64, 4, 104 * K, 2>());
    }
}

// Where things lie in the workspace of the tensor-core kernels.
struct Layout {
    size_t yp, count, taken, bytes;
};
template <typename T> static int slots_of(i64 tokens, i64 E, i64 k) {
    return (int)(slot_is_expert<T>(tokens, E, k) ? E : std::min(E, tokens * k));
}
template <typename Ty> static Layout layout(Context* c, i64 T, i64 hidden, i64 mid, i64 E, i64 k) {
    Layout l{};
    const int slots = slots_of<Ty>(T, E, k);
    with_shape<Ty>(c, T, hidden, mid, E, k, [&](auto shape) {
        using P = decltype(shape);
        const Plan d = plan(c, slots, (int)T, false, (int)mid, (int)hidden, P::BD, P::PD);
        l.yp = align256((size_t)T * k * mid * sizeof(Ty));
        l.count = l.yp + align256((size_t)d.grid.y * T * k * hidden * 4);
        l.taken = l.count + align256((size_t)cdiv(hidden, P::BD) * T * 4);
        l.bytes = l.taken + align256((size_t)T * (k + 1) * 4);
    });
    return l;
}

template <typename T> static void run_tc(Context* c, TcArgs a, const void* w1, const void* w3, const void* w2) {
    const int slots = slots_of<T>(a.T, a.E, a.k);
    with_shape<T>(c, a.T, a.hidden, a.mid, a.E, a.k, [&](auto shape) {
        using P = decltype(shape);
        using U = Tc<T, P::ALL, 2, P::NT, P::BU, P::CU, P::RU>;
        using D = Tc<T, P::ALL, 1, P::NT, P::BD, P::CD, P::RD>;
        // found first, the experts are found twice, and by the same sums: their order goes by the number of warps
        static_assert(P::ALL || P::CU == P::CD, "both kernels must choose the same experts to the last bit");
        const int dt = sizeof(T) == 4 ? CATNN_F32 : CATNN_BF16;
        const CUtensorMap m1 = tma_map_stack(w1, a.E, a.hidden, a.mid, dt, U::BOX, BK);
        const CUtensorMap m3 = tma_map_stack(w3, a.E, a.hidden, a.mid, dt, U::BOX, BK);
        const CUtensorMap m2 = tma_map_stack(w2, a.E, a.mid, a.hidden, dt, D::BOX, BK);
        const Plan u = plan(c, slots, a.T, true, a.hidden, a.mid, P::BU, P::PU);
        const Plan d = plan(c, slots, a.T, false, a.mid, a.hidden, P::BD, P::PD);
        a.up_run = u.run;
        a.down_run = d.run;
        a.counts = cdiv(a.hidden, P::BD) * a.T;
        launch(c, k_up_tc<T, P::ALL, P::NT, P::BU, P::CU, P::RU, P::PU>, U::THREADS, u.grid, u.cluster, U::smem(a.T, a.k), false, a,
               m1, m3);
        launch(c, k_down_tc<T, P::ALL, P::NT, P::BD, P::CD, P::RD, P::PD>, D::THREADS, d.grid, d.cluster, D::smem(a.T, a.k), true, a,
               m2);
    });
}

}  // namespace few

using namespace few;

// Large enough for either form: which one runs hangs on the pointers' alignment too.
size_t moe_few_workspace(Context* c, i64 T, i64 hidden, i64 mid, i64 E, i64 k, int dtype) {
    if (T == 0) return 0;
    const size_t plain = (size_t)T * k * mid * sizeof(float);
    return std::max(plain, dtype == CATNN_BF16 ? layout<bf16>(c, T, hidden, mid, E, k).bytes
                                               : layout<float>(c, T, hidden, mid, E, k).bytes);
}

template <typename Ty>
static void moe_few_tc(Context* c, const void* x, const void* gate, const void* w1, const void* w3, const void* w2, void* y, i64 T,
                       i64 hidden, i64 mid, i64 E, i64 k, void* work) {
    const Layout l = layout<Ty>(c, T, hidden, mid, E, k);
    char* at = (char*)work;
    run_tc<Ty>(c,
               {x, gate, work, y, (float*)(at + l.yp), (unsigned*)(at + l.taken), (unsigned*)(at + l.count),
                c->status + FEW_STATUS_SLOT, c->few_patience, (int)T, (int)hidden, (int)mid, (int)E, (int)k, 0, 0, 0},
               w1, w3, w2);
}

void moe_few(Context* c, const void* x, const void* gate, const void* w1, const void* w3, const void* w2, void* y, i64 T,
             i64 hidden, i64 mid, i64 E, i64 k, int dtype, void* work) {
    if (T == 0) return;
    const auto al = [](const void* p) { return aligned_to(p, 16); };
    const int piece = dtype == CATNN_BF16 ? 8 : 4;
    if (hidden % piece == 0 && mid % piece == 0 && hidden >= BK && mid >= BK && al(x) && al(gate) && al(w1) && al(w3) && al(w2) &&
        al(y)) {
        if (dtype == CATNN_BF16) moe_few_tc<bf16>(c, x, gate, w1, w3, w2, y, T, hidden, mid, E, k, work);
        else moe_few_tc<float>(c, x, gate, w1, w3, w2, y, T, hidden, mid, E, k, work);
        return;
    }
    Args a{x, gate, w1, w3, w2, y, (float*)work, (int)T, (int)hidden, (int)mid, (int)E, (int)k};
    const dim3 up(cdiv(mid, THREADS), (unsigned)T), down(cdiv(hidden, THREADS), (unsigned)T);
    if (dtype == CATNN_BF16) {
        k_up_any<bf16><<<up, THREADS, 0, c->stream>>>(a);
        k_down_any<bf16><<<down, THREADS, 0, c->stream>>>(a);
    } else {
        k_up_any<float><<<up, THREADS, 0, c->stream>>>(a);
        k_down_any<float><<<down, THREADS, 0, c->stream>>>(a);
    }
    launched(c, 2);
}

}  // namespace catnn
