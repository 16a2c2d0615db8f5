// Attention of one new token of each sequence against a paged cache:
//   o = softmax(q·Kᵀ/√hd)·V over the sequence's last min(len, window)
//   positions, lse = log Σ exp of the scaled scores.
// Position j of sequence b lies in slot j % page of the pool's page
// table[b][j / page]; a page is [Hkv, page, hd], so that one head's keys of a
// page are one run of memory.
#include <algorithm>

#include "ops.cuh"
#include "paged_place.cuh"

namespace catnn {
namespace paged {

constexpr int MAX_HD = 128;

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
};

constexpr int WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) k_paged(const __grid_constant__ Args a) {
    __shared__ float sm[WARPS], sl[WARPS], so[WARPS][MAX_HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const i64 b = blockIdx.x / a.h;
    const int head = (int)(blockIdx.x - b * a.h), kvh = head / (a.h / a.hkv);
    const i64 held = (i64)a.max_pages * a.page;
    i64 len = a.lens[b];
    if (len > held) {
        if (a.err) atomicExch(a.err, 1);
        len = held;
    }
    const i64 first = a.window > 0 && len > a.window ? len - a.window : 0;
    float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int d = lane + 32 * u;
        q[u] = d < a.hd ? ld((const T*)a.q + b * a.q_stride + (i64)head * a.hd + d) * a.scale : 0.f;
    }
    for (i64 j = first + warp; j < len; j += WARPS) {
        i64 row = place::cache_index(a.table, b, (int)j, a.page, a.max_pages, a.pages, a.hkv, a.hd);
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
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float keep = expf(m - mn), p = expf(s - mn);
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
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += sl[w] != 0.f ? sl[w] * expf(sm[w] - top) : 0.f;
    for (int d = threadIdx.x; d < a.hd; d += WARPS * 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += sl[w] != 0.f ? so[w][d] * expf(sm[w] - top) : 0.f;
        st((T*)a.o + (b * a.h + head) * a.hd + d, total != 0.f ? v / total : 0.f);
    }
    if (threadIdx.x == 0) a.lse[b * a.h + head] = total != 0.f ? top + logf(total) : -INFINITY;
}

}  // namespace paged

using namespace paged;

size_t paged_attention_workspace(Context*, i64, i64, i64, i64) { return 0; }

void paged_attention(Context* c, const void* q, i64 q_stride, const void* kc, const void* vc, const int32_t* table,
                     const int32_t* lens, void* o, float* lse, i64 seqs, i64 h, i64 hkv, i64 hd, i64 pages, i64 page,
                     i64 max_pages, i64 window, int dtype, void*, int* err) {
    if (seqs == 0) return;
    Args a{q, kc, vc, o, lse, table, lens, seqs, (int)h, (int)hkv, (int)hd, (int)page, (int)max_pages, (int)window, pages,
           q_stride, 1.0f / sqrtf((float)hd), err};
    if (dtype == CATNN_BF16) k_paged<bf16><<<(int)(seqs * h), WARPS * 32, 0, c->stream>>>(a);
    else k_paged<float><<<(int)(seqs * h), WARPS * 32, 0, c->stream>>>(a);
    launched(c);
}

}  // namespace catnn
