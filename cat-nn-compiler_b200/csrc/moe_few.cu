// A whole mixture-of-experts layer for a few tokens (at most 64):
//   logits = x·gate; the k largest, ties to the lower index; w = softmax
//   over those k; y = Σ_j w_j·(silu(x·w1)·(x·w3))·w2 of the j-th expert.
// The grouped GEMMs of the block for many tokens pad every expert to 128
// rows and take nine launches; here two kernels read the chosen experts'
// weights once: the first routes and forms h, the second routes again (from
// x and gate, cheaper than a third launch) and forms y.
#include <algorithm>

#include "ops.cuh"

namespace catnn {
namespace few {

constexpr int MAX_E = 32;
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

}  // namespace few

using namespace few;

size_t moe_few_workspace(Context*, i64 T, i64, i64 mid, i64, i64 k, int) { return (size_t)T * k * mid * sizeof(float); }

void moe_few(Context* c, const void* x, const void* gate, const void* w1, const void* w3, const void* w2, void* y, i64 T,
             i64 hidden, i64 mid, i64 E, i64 k, int dtype, void* work) {
    if (T == 0) return;
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
