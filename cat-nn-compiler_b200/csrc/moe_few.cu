// A whole mixture-of-experts layer for a few tokens (at most 64):
//   logits = x·gate; the k largest, ties to the lower index; w = softmax
//   over those k; y = Σ_j w_j·(silu(x·w1)·(x·w3))·w2 of the j-th expert.
// The grouped GEMMs of the block for many tokens pad every expert to 128
// rows and take nine launches; here two kernels read the chosen experts'
// weights once: the first routes and forms h, the second routes again (from
// x and gate, cheaper than a third launch) and forms y.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

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
// Of up to 16 tokens the experts that any token takes are found first, by
// every CTA of both kernels for itself (ALL = false): a slot of the grid is the
// slot-th of them. Of more tokens (nearly) every expert has some: a slot is an
// expert, whose first tiles are fetched while the first kernel routes, and
// the second kernel, whose first tiles are fetched beside the first's last,
// reads what the first found (ALL = true).
constexpr int BK = 64, XPITCH = 144;
constexpr int SMEM_MAX = 128 * 1024;  // the widest ring and what lies beside it

struct TcArgs {
    const bf16 *x, *gate;
    bf16 *h, *y;
    float* yp;        // [runs][T·k, hidden]: each pair's share of y from each run of rows, before its weight
    unsigned* taken;  // [T], then [T·k] weights: what the first kernel found (ALL)
    unsigned* count;  // [column tiles of hidden]: CTAs that have put theirs there
    int* status;
    int T, hidden, mid, E, k;
    int up_run, down_run;  // rows of a matrix that one CTA takes
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

// `issued` is called by every warp when its first batch's loads are on their way.
template <int R8, int CW, typename Issued>
__device__ __forceinline__ void logits_tc(const TcArgs& a, int t0, int rows, char* gs, float* part, Issued issued) {
    constexpr int NB = R8 == 1 ? 8 : 4;  // runs of 32 k in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, kj = (lane & 3) * 8;
    const int nt = (a.E + 7) / 8, ep = nt * 8;
    gs += warp * NB * 512;
    const uint32_t gaddr = tc::smem_u32(gs) + (8 * ((lane & 7) >> 1) + (lane & 1) + 2 * (lane >> 3)) * 16;
    const bf16* xrow[R8];
#pragma unroll
    for (int i = 0; i < R8; ++i) xrow[i] = a.x + (i64)(t0 + min(i * 8 + row, rows - 1)) * a.hidden + kj;  // a row past the last is not used
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
            const bf16* grow = a.gate + (i64)(k0 + lane) * a.E + j * 8;
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
template <int R8, int CW, typename Prefetch>
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
    } else if (rows > 0 && warp * 32 < a.hidden) {
        logits_tc<R8, CW>(a, t0, rows, room + CW * RT * MAX_E * 4, part, issued);
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
        const unsigned taken = choose(l, a.E, a.k, lane, top);
        const int t = t0 + i;
        if (lane < copies) to[t] = taken;
        if (w_here || tell) {
            const bool in = taken >> lane & 1u;
            float w = in ? __expf(l - top) : 0.f;
            w = __fdividef(w, fmaxf(warp_sum(w), 1e-30f));
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
template <bool ALL, int M, int NT, int BN_, int CW, int ROOM> struct Tc {
    static constexpr int BN = BN_, BOX = BN < 64 ? BN : 64, THREADS = (CW + 1) * 32;
    static constexpr int KG = CW * 16 / BN;  // groups of warps that share a tile's columns and split its k
    static constexpr int W_BYTES = M * BK * BN * 2, RED_PITCH = BN + 4;  // bytes; floats
    static constexpr int RED = M * NT * 8 * RED_PITCH;                   // floats of one group's sums
    static constexpr int MIN_STAGES = ROOM / (W_BYTES + NT * 8 * XPITCH);
    static constexpr int PRE = ALL ? (MIN_STAGES < 3 ? MIN_STAGES : 3) : 0;  // stages filled before routing
    static constexpr int SCRATCH = CW * (RT * MAX_E * 4 + (NT == 1 ? 8 : 4) * 512);
    static_assert(ROOM % 1024 == 0 && MIN_STAGES >= 2, "two stages at least");
    static_assert(KG * RED * 4 <= ROOM && (M == 1 && ALL ? 0 : PRE * W_BYTES + SCRATCH) <= ROOM,
                  "the parts, and routing beside the first stages, lie in the ring");
    static_assert(1024 + ROOM + 2 * MAX_STAGES * 8 + MAX_T * (8 + 4 * MAX_E) <= SMEM_MAX, "smem()'s largest");
    static size_t smem(int T, int k) { return 1024 + ROOM + 2 * MAX_STAGES * 8 + routes_bytes(T, k); }

    char* ring;
    uint64_t *full, *empty;
    const CUtensorMap* w[2];
    int r0, r1, col0, iters;

    __device__ __forceinline__ Tc(const TcArgs& a, char* raw, Routes& r, const CUtensorMap* w0, const CUtensorMap* w1, int run,
                                  int rows, int cols) {
        ring = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
        full = (uint64_t*)(ring + ROOM);
        empty = full + MAX_STAGES;
        r.taken = (unsigned*)(empty + MAX_STAGES);
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
                tc::tma_load_3d(at + (m * BN + c) * BK * 2, w[m], col0 + c, r0 + it * BK, expert, &full[st]);
    }
    // An expert that no token takes: let what was fetched land, then leave.
    __device__ __forceinline__ void drain(const TcArgs& a) const {
        if (threadIdx.x >= CW * 32)
            for (int it = 0; it < PRE && it < iters; ++it) {
                tc::mbar_arrive(&full[it]);
                tc::mbar_wait(&full[it], 0, a.status, 4, 4000000000ll, false);
            }
    }
};

// Rows [r0, r1) of the expert's matrices times the same columns of `rows`
// (row index `idx`, row length `len`), left in shared memory: sum(m, token
// index, column in the tile).
template <bool ALL, int M, int NT, int BN, int CW, int ROOM, typename Wait>
__device__ __forceinline__ void product(const Tc<ALL, M, NT, BN, CW, ROOM>& s, const TcArgs& a, const Routes& r, const short* idx,
                                        const bf16* rows, int len, Wait wait) {
    using S = Tc<ALL, M, NT, BN, CW, ROOM>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int iters = s.iters, nte = (r.n + 7) / 8, xbytes = nte * 8 * XPITCH;
    const int stages = min(MAX_STAGES, ROOM / (S::W_BYTES + xbytes));
    char* const xring = s.ring + stages * S::W_BYTES;
    float acc[M][NT][4];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[m][j][u] = 0.f;
    if (warp == CW) {
        auto tokens = [&](int it, int st) {
            const uint32_t at = tc::smem_u32(xring + st * xbytes);
            const int k0 = s.r0 + it * BK, chunks = (min(s.r1, k0 + BK) - k0) >> 3;  // of 8 k
            for (int i = lane; i < r.n * 8; i += 32) {
                const int row = i >> 3, c = i & 7;
                const bool on = c < chunks;
                tc::cp_async16(at + row * XPITCH + c * 16, rows + (i64)idx[row] * len + (on ? k0 + c * 8 : 0), on);
            }
            tc::cp_async_arrive(&s.full[st]);
        };
        // weights first: they wait for nobody
        if (lane == 0)
            for (int it = S::PRE; it < iters && it < stages; ++it) s.weights(it, it, r.expert);
        __syncwarp();
        wait();
        for (int it = 0; it < iters && it < stages; ++it) tokens(it, it);
        for (int it = stages, st = 0, ph = 0; it < iters; ++it) {
            tc::mbar_wait(&s.empty[st], ph, a.status, 4, 4000000000ll, false);
            if (lane == 0) s.weights(it, st, r.expert);
            __syncwarp();
            tokens(it, st);
            if (++st == stages) st = 0, ph ^= 1;
        }
    } else {
        wait();
        const int k8 = lane & 7, hi = lane >> 4 & 1, mid8 = lane >> 3 & 1;
        const int wm = warp % (BN / 16), kg = warp / (BN / 16);
        const uint32_t wcol = wm / (S::BOX / 16) * (BK * S::BOX * 2), chunk = wm % (S::BOX / 16) * 2 + mid8;
        for (int it = 0, st = 0, ph = 0; it < iters; ++it) {
            const int kk = min(BK, s.r1 - s.r0 - it * BK);
            tc::mbar_wait(&s.full[st], ph, a.status, 4, 4000000000ll, false);
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
                    tc::ldsm4(b, xb + (j * 8 + k8) * XPITCH + (k0 / 8 + (lane >> 3)) * 16);
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
    __syncthreads();  // every tile of the ring has landed and been read
    if (warp < CW) {
        const int wm = warp % (BN / 16), kg = warp / (BN / 16);
        float* red = (float*)s.ring + kg * S::RED + wm * 16 + (lane >> 2) + (lane & 3) * 2 * S::RED_PITCH;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (j >= nte) break;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    red[(m * NT * 8 + j * 8 + (u & 1)) * S::RED_PITCH + (u >> 1) * 8] = acc[m][j][u];
            }
    }
}

// Adds to v[m] four columns of token t of one CTA's sums.
template <typename S, int M, int NT> __device__ __forceinline__ void add_sums(const float* red, int t, int c, float4 (&v)[M]) {
#pragma unroll
    for (int g = 0; g < S::KG; ++g)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const float4 w = *(const float4*)(red + g * S::RED + (m * NT * 8 + t) * S::RED_PITCH + c);
            v[m].x += w.x;
            v[m].y += w.y;
            v[m].z += w.z;
            v[m].w += w.w;
        }
}

template <bool ALL, int NT, int BN, int CW, int ROOM, int PER_SM>
__global__ void __launch_bounds__((CW + 1) * 32, PER_SM)
    k_up_tc(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap w1, const __grid_constant__ CUtensorMap w3) {
    extern __shared__ char raw[];
    tc::launch_dependents();  // the second kernel may take the SMs' free places and fetch w2
    Routes r;
    using S = Tc<ALL, 2, NT, BN, CW, ROOM>;
    const S s(a, raw, r, &w1, &w3, a.up_run, a.hidden, a.mid);
    const bool first = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
    if (first)
        for (int i = threadIdx.x; i < (a.hidden + 63) / 64; i += S::THREADS) a.count[i] = 0u;
    route_tc<NT == 1 ? 1 : 2, CW>(a, s.ring + S::PRE * S::W_BYTES, r, nullptr,
                                  ALL && blockIdx.x < cg::this_cluster().dim_blocks().x && blockIdx.z == 0, [&] { s.prefetch(); });
    find_expert<ALL, CW>(a, blockIdx.z, r);
    if (r.n == 0) {  // the whole cluster: it shares its slot
        s.drain(a);
        return;
    }
    __syncthreads();
    product(s, a, r, r.tok, a.x, a.hidden, [] {});
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
            add_sums<S, 2, NT>(runs > 1 ? cl.map_shared_rank((float*)s.ring, p * cx + ix) : (float*)s.ring, t, c, v);
        const float* u = (const float*)&v[0];
        const float* g = (const float*)&v[1];
        float h[4];
        // held in bf16, the type that the second product multiplies in
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = u[j] / (1.f + __expf(-u[j])) * g[j];
        stv<bf16, 4>(a.h + (i64)r.pair[t] * a.mid + s.col0 + c, h);
    }
    if (runs > 1) cl.sync();  // no CTA leaves while another reads its sums
}

template <bool ALL, int NT, int BN, int CW, int ROOM, int PER_SM>
__global__ void __launch_bounds__((CW + 1) * 32, PER_SM)
    k_down_tc(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap w2) {
    extern __shared__ char raw[];
    __shared__ bool last;
    Routes r;
    using S = Tc<ALL, 1, NT, BN, CW, ROOM>;
    const S s(a, raw, r, &w2, &w2, a.down_run, a.mid, a.hidden);
    if (ALL) {
        s.prefetch();
        tc::grid_dependency_wait();
        for (int i = threadIdx.x; i < a.T * (a.k + 1); i += S::THREADS) r.taken[i] = __ldcg(a.taken + i);
        __syncthreads();
    } else {
        route_tc<NT == 1 ? 1 : 2, CW>(a, s.ring, r, r.w, false, [] {});
    }
    find_expert<ALL, CW>(a, blockIdx.z, r);
    if (r.n == 0) {
        s.drain(a);
        return;
    }
    __syncthreads();
    const int col0 = s.col0;
    product(s, a, r, r.pair, a.h, a.mid, [] { if (!ALL) tc::grid_dependency_wait(); });
    __syncthreads();
    const i64 run_size = (i64)a.T * a.k * a.hidden;
#pragma unroll 1
    for (int i = threadIdx.x; i < r.n * (BN / 4); i += S::THREADS) {
        const int t = i / (BN / 4), c = (i - t * (BN / 4)) * 4;
        if (col0 + c >= a.hidden) continue;
        float4 v[1] = {make_float4(0.f, 0.f, 0.f, 0.f)};
        add_sums<S, 1, NT>((float*)s.ring, t, c, v);
        *(float4*)(a.yp + blockIdx.y * run_size + (i64)r.pair[t] * a.hidden + col0 + c) = v[0];
    }
    // the last CTA of a column tile adds up what the tokens' experts gave, expert by expert and run by run
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.count + blockIdx.x, 1u) == (unsigned)r.active * gridDim.y - 1u;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // four tokens at a time, so that their loads are in flight together
    constexpr int Q = BN / 4, AT_ONCE = 4;
    const int c = col0 + threadIdx.x % Q * 4;
    if (c >= a.hidden) return;
#pragma unroll 1
    for (int tb = threadIdx.x / Q; tb < a.T; tb += S::THREADS / Q * AT_ONCE) {
        float4 y[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int j = 0; j < a.k; ++j) {
            float4 v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int q = 0; q < (int)gridDim.y; ++q)
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int t = min(tb + i * (S::THREADS / Q), a.T - 1);
                    const float4 u = __ldcg((const float4*)(a.yp + q * run_size + ((i64)t * a.k + j) * a.hidden + c));
                    v[i].x += u.x;
                    v[i].y += u.y;
                    v[i].z += u.z;
                    v[i].w += u.w;
                }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float w = r.w[min(tb + i * (S::THREADS / Q), a.T - 1) * a.k + j];
                y[i].x = fmaf(w, v[i].x, y[i].x);
                y[i].y = fmaf(w, v[i].y, y[i].y);
                y[i].z = fmaf(w, v[i].z, y[i].z);
                y[i].w = fmaf(w, v[i].w, y[i].w);
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int t = tb + i * (S::THREADS / Q);
            const float o[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
            if (t < a.T) stv<bf16, 4>(a.y + (i64)t * a.hidden + c, o);
        }
    }
}

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// How many runs a matrix's rows are cut into (at most 8, a cluster): as many
// as the SMs hold CTAs at once, of at least two tiles each; with all of them
// resident they share the memory evenly and end together.
static int runs_of(Context* c, i64 tiles, i64 rows, int per_sm) {
    int s = 1;
    while (s < 8 && tiles * 2 * s <= (i64)c->sm_count * per_sm && rows / (2 * s) >= 2 * BK) s *= 2;
    return s;
}

template <typename Kern, typename... A>
static void launch(Context* c, Kern k, int threads, dim3 grid, dim3 cluster, size_t smem, bool dependent, const A&... args) {
    // a function's limit on one device holds from then on; `Kern` is the same type for several kernels
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> raised;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (raised.insert({(const void*)k, c->device}).second) {
            CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
            // all of the SM's memory as shared: the second kernel's CTAs come to SMs that the first still holds
            CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        }
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

// f(Shape) for a problem.
template <typename F> static void with_shape(Context* c, i64 T, i64 mid, i64 slots, F f) {
    const bool thin = (i64)cdiv(mid, 32) * slots <= (i64)c->sm_count * 4;
    if (T <= 8 && thin) f(Shape<false, 1, 32, 4, 52 * K, 2, 64, 4, 52 * K, 3>());
    else if (T <= 8) f(Shape<false, 1, 64, 4, 52 * K, 4, 64, 4, 52 * K, 4>());
    else if (T <= 16 && thin) f(Shape<false, 2, 32, 4, 52 * K, 2, 64, 4, 52 * K, 3>());
    else if (T <= 16) f(Shape<false, 2, 64, 4, 52 * K, 4, 64, 4, 52 * K, 4>());
    else if (T <= 32) f(Shape<true, 4, 128, 8, 104 * K, 2, 64, 4, 104 * K, 2>());
    else f(Shape<true, 8, 128, 8, 104 * K, 2, 64, 4, 104 * K, 2>());
}

// Where things lie in the workspace of the tensor-core kernels.
struct Layout {
    size_t yp, count, taken, bytes;
};
static int slots_of(i64 T, i64 E, i64 k) { return (int)(T > 16 ? E : std::min(E, T * k)); }
static Layout layout(Context* c, i64 T, i64 hidden, i64 mid, i64 E, i64 k) {
    Layout l{};
    const int slots = slots_of(T, E, k);
    with_shape(c, T, mid, slots, [&](auto shape) {
        using P = decltype(shape);
        const Plan d = plan(c, slots, (int)T, false, (int)mid, (int)hidden, P::BD, P::PD);
        l.yp = align256((size_t)T * k * mid * 2);
        l.count = l.yp + align256((size_t)d.grid.y * T * k * hidden * 4);
        l.taken = l.count + align256((size_t)cdiv(hidden, 64) * 4);
        l.bytes = l.taken + align256((size_t)T * (k + 1) * 4);
    });
    return l;
}

static void run_tc(Context* c, TcArgs a, const void* w1, const void* w3, const void* w2) {
    const int slots = slots_of(a.T, a.E, a.k);
    with_shape(c, a.T, a.mid, slots, [&](auto shape) {
        using P = decltype(shape);
        const CUtensorMap m1 = tma_map_stack(w1, a.E, a.hidden, a.mid, CATNN_BF16, std::min(64, P::BU), BK);
        const CUtensorMap m3 = tma_map_stack(w3, a.E, a.hidden, a.mid, CATNN_BF16, std::min(64, P::BU), BK);
        const CUtensorMap m2 = tma_map_stack(w2, a.E, a.mid, a.hidden, CATNN_BF16, std::min(64, P::BD), BK);
        const Plan u = plan(c, slots, a.T, true, a.hidden, a.mid, P::BU, P::PU);
        const Plan d = plan(c, slots, a.T, false, a.mid, a.hidden, P::BD, P::PD);
        a.up_run = u.run;
        a.down_run = d.run;
        launch(c, k_up_tc<P::ALL, P::NT, P::BU, P::CU, P::RU, P::PU>, (P::CU + 1) * 32, u.grid, u.cluster,
               Tc<P::ALL, 2, P::NT, P::BU, P::CU, P::RU>::smem(a.T, a.k), false, a, m1, m3);
        launch(c, k_down_tc<P::ALL, P::NT, P::BD, P::CD, P::RD, P::PD>, (P::CD + 1) * 32, d.grid, d.cluster,
               Tc<P::ALL, 1, P::NT, P::BD, P::CD, P::RD>::smem(a.T, a.k), true, a, m2);
    });
}

}  // namespace few

using namespace few;

// Large enough for either form: which one runs hangs on the pointers' alignment too.
size_t moe_few_workspace(Context* c, i64 T, i64 hidden, i64 mid, i64 E, i64 k, int dtype) {
    if (T == 0) return 0;
    const size_t plain = (size_t)T * k * mid * sizeof(float);
    return dtype == CATNN_BF16 ? std::max(plain, layout(c, T, hidden, mid, E, k).bytes) : plain;
}

void moe_few(Context* c, const void* x, const void* gate, const void* w1, const void* w3, const void* w2, void* y, i64 T,
             i64 hidden, i64 mid, i64 E, i64 k, int dtype, void* work) {
    if (T == 0) return;
    const auto al = [](const void* p) { return aligned_to(p, 16); };
    if (dtype == CATNN_BF16 && hidden % 8 == 0 && mid % 8 == 0 && hidden >= BK && mid >= BK && al(x) && al(gate) && al(w1) &&
        al(w3) && al(w2) && al(y)) {
        const Layout l = layout(c, T, hidden, mid, E, k);
        char* at = (char*)work;
        run_tc(c,
               {(const bf16*)x, (const bf16*)gate, (bf16*)work, (bf16*)y, (float*)(at + l.yp), (unsigned*)(at + l.taken),
                (unsigned*)(at + l.count), c->status, (int)T, (int)hidden, (int)mid, (int)E, (int)k, 0, 0},
               w1, w3, w2);
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
