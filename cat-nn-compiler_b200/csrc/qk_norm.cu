// RMS norm of every query and key head with the position rotation in the
// same pass (forward and adjoint), and the append of new keys and values to
// a paged cache with both applied on the way.
//
// With x one head's row of hd values, r = (mean(x²) + eps)^(-1/2) and R(p)
// the rotation of the pairs (2i, 2i+1) by p·θ^(-2i/hd):
//   forward  y = R(p)·(x·r·w)
//   adjoint  g = R(p)ᵀ·dy, x̂ = x·r, dw = Σ_rows g·x̂,
//            dx = r·(g·w − x̂·mean(g·w·x̂))
// Every kernel reads its rows once and writes them once, so HBM bounds them.
//
// A row is held by the smallest power-of-two group of lanes that takes it in
// 16-byte pieces (8 bf16 or 4 fp32 values a lane; hd 80 and 96 leave lanes
// idle), so its sums are shuffles within the group, and a lane keeps the same
// pairs for all heads of a token: their sines are taken once per token.
// Rows that are not 16-byte aligned take one element pair a lane instead.
#include <algorithm>
#include <cmath>

#include "ops.cuh"
#include "paged_place.cuh"
#include "tc_prims.cuh"

namespace catnn {
namespace qkn {

constexpr int MAX_HD = 256;
constexpr int WARPS = 8;

// θ^(-2i/hd) / 2π: the pair's turns per position, in f64 because a far
// position times a rounded f32 frequency is off by whole radians.
struct Freq {
    double turn[MAX_HD / 2];
};

static const Freq& freq_of(Context* c, i64 hd, double theta) {
    // kept per context as plain host values: a captured graph carries its own copy in the kernel's arguments
    static_assert(sizeof(Freq) <= sizeof(c->turns), "Context::turns holds the widest head");
    if (c->turns_hd != hd || c->turns_theta != theta) {
        const double two_pi = 6.283185307179586476925286766559;
        for (i64 i = 0; i < hd / 2; ++i) c->turns[i] = std::pow(theta, -2.0 * (double)i / (double)hd) / two_pi;
        c->turns_hd = hd;
        c->turns_theta = theta;
    }
    return *reinterpret_cast<const Freq*>(c->turns);
}

// (cos, sin) of the angle pos·turn·2π. The turns are reduced to [-1/2, 1/2]
// in f64, where what is left is exact to 2^-53·|turns|. fp32 rows take
// sincospi (2 ulp); bf16 rows the hardware sine, whose error of 2^-21 is far
// below the 2^-9 of the rounding that follows.
template <typename T> __device__ __forceinline__ float2 cos_sin(int pos, double turn) {
    double t = (double)pos * turn;
    t -= rint(t);
    float s, c;
    if constexpr (sizeof(T) == 4) sincospif(2.f * (float)t, &s, &c);
    else __sincosf(6.28318530717958648f * (float)t, &s, &c);
    return make_float2(c, s);
}

template <int LPH> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);

template <int V> __device__ __forceinline__ void rotate(float (&x)[V], const float2 (&cs)[V / 2]) {
#pragma unroll
    for (int u = 0; u < V / 2; ++u) {
        float a = x[2 * u], b = x[2 * u + 1];
        x[2 * u] = a * cs[u].x - b * cs[u].y;
        x[2 * u + 1] = a * cs[u].y + b * cs[u].x;
    }
}

struct FwdArgs {
    const void *q, *k;
    i64 q_stride, k_stride;  // elements between tokens
    const float *wq, *wk;
    const int32_t* pos;  // [tokens], or null: token % s
    void *qo, *ko;
    i64 tokens, s;
    int h, hkv, hd;
    float eps;
    // a unit is up to `per` row groups of a token, `units` units a token
    int per, units;
};

// 16 bytes as V values.
template <typename T, int V> __device__ __forceinline__ void unpack(const uint4& r, float (&o)[V]) {
    if constexpr (sizeof(T) == 4) {
        o[0] = __uint_as_float(r.x), o[1] = __uint_as_float(r.y), o[2] = __uint_as_float(r.z), o[3] = __uint_as_float(r.w);
    } else {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[2 * j] = __uint_as_float(w[j] << 16);
            o[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
}

// Forward on 16-byte pieces. Group g of a token holds heads
// [g·HPW, (g+1)·HPW) of its H query heads followed by its Hkv key heads. A
// warp walks the units in grid order; all rows of a unit are on their way
// before its sines are taken.
constexpr int UNIT = 6;  // row groups of a unit, at most
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 3) k_qk_fwd(const __grid_constant__ FwdArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, HPW = 32 / LPH;
    const int lane = threadIdx.x & 31, sub = lane / LPH, li = lane % LPH, e0 = li * V, heads = a.h + a.hkv;
    const bool in = e0 < a.hd;
    float wq[V], wk[V];
#pragma unroll
    for (int u = 0; u < V; ++u) wq[u] = wk[u] = 0.f;
    if (in) {
        ldv<float, V>(a.wq + e0, wq);
        ldv<float, V>(a.wk + e0, wk);
    }
    const i64 all = a.tokens * a.units;
    for (i64 unit = (i64)blockIdx.x * WARPS + (threadIdx.x >> 5); unit < all; unit += (i64)gridDim.x * WARPS) {
        const i64 tok = a.units == 1 ? unit : unit / a.units;
        const int head0 = (int)(unit - tok * a.units) * a.per * HPW + sub;
        const T* qrow = (const T*)a.q + tok * a.q_stride + e0;
        const T* krow = (const T*)a.k + tok * a.k_stride + e0;
        uint4 raw[UNIT];
#pragma unroll
        for (int g = 0; g < UNIT; ++g) {
            const int head = head0 + g * HPW;
            raw[g] = make_uint4(0, 0, 0, 0);
            if (g < a.per && in && head < heads)
                raw[g] = *(const uint4*)(head < a.h ? qrow + (i64)head * a.hd : krow + (i64)(head - a.h) * a.hd);
        }
        const int p = a.pos ? a.pos[tok] : (int)(tok % a.s);
        float2 cs[V / 2];
        if (in)
#pragma unroll
            for (int u = 0; u < V / 2; ++u) cs[u] = cos_sin<T>(p, f.turn[li * (V / 2) + u]);
        T* qo = (T*)a.qo + tok * a.h * a.hd + e0;
        T* ko = (T*)a.ko + tok * a.hkv * a.hd + e0;
#pragma unroll
        for (int g = 0; g < UNIT; ++g) {
            if (g >= a.per) break;
            const int head = head0 + g * HPW;
            const bool isq = head < a.h;
            float x[V];
            unpack<T, V>(raw[g], x);
            float ss = 0.f;
#pragma unroll
            for (int u = 0; u < V; ++u) ss = fmaf(x[u], x[u], ss);
            const float r = rsqrtf(group_sum<LPH>(ss) / (float)a.hd + a.eps);
            if (!in || head >= heads) continue;
#pragma unroll
            for (int u = 0; u < V; ++u) x[u] = x[u] * r * (isq ? wq[u] : wk[u]);
            rotate<V>(x, cs);
            stv<T, V>(isq ? qo + (i64)head * a.hd : ko + (i64)(head - a.h) * a.hd, x);
        }
    }
}

// Any even hd and any alignment: a warp to a row, lane l holding the pairs
// l, l + 32, …
constexpr int PAIRS = MAX_HD / 64;
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) k_qk_fwd_any(const __grid_constant__ FwdArgs a, const __grid_constant__ Freq f) {
    const int lane = threadIdx.x & 31, heads = a.h + a.hkv;
    const i64 row = (i64)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const i64 tok = row / heads;
    if (tok >= a.tokens) return;
    const int head = (int)(row - tok * heads);
    const bool isq = head < a.h;
    const T* x = isq ? (const T*)a.q + tok * a.q_stride + (i64)head * a.hd
                     : (const T*)a.k + tok * a.k_stride + (i64)(head - a.h) * a.hd;
    T* y = isq ? (T*)a.qo + (tok * a.h + head) * a.hd : (T*)a.ko + (tok * a.hkv + head - a.h) * a.hd;
    const float* w = isq ? a.wq : a.wk;
    const int p = a.pos ? a.pos[tok] : (int)(tok % a.s);
    float v[2 * PAIRS], ss = 0.f;
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        const int i = lane + 32 * u;
        v[2 * u] = v[2 * u + 1] = 0.f;
        if (i < a.hd / 2) {
            v[2 * u] = ld(x + 2 * i);
            v[2 * u + 1] = ld(x + 2 * i + 1);
        }
        ss = fmaf(v[2 * u], v[2 * u], fmaf(v[2 * u + 1], v[2 * u + 1], ss));
    }
    const float r = rsqrtf(warp_sum(ss) / (float)a.hd + a.eps);
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        const int i = lane + 32 * u;
        if (i >= a.hd / 2) continue;
        const float2 cs = cos_sin<T>(p, f.turn[i]);
        const float x0 = v[2 * u] * r * w[2 * i], x1 = v[2 * u + 1] * r * w[2 * i + 1];
        st(y + 2 * i, x0 * cs.x - x1 * cs.y);
        st(y + 2 * i + 1, x0 * cs.y + x1 * cs.x);
    }
}

struct BwdArgs {
    const void *q, *k, *gq, *gk;
    i64 q_stride, k_stride, gq_stride, gk_stride;
    const float *wq, *wk;
    const int32_t* pos;
    void *dq, *dk;
    float* part;  // a row of hd sums from each CTA: those of wq, then those of wk
    i64 tokens, s;
    int h, hkv, hd;
    float eps;
    int per[2], units[2];  // groups of a unit and units of a token, of queries and of keys
    int q_ctas;            // CTAs that have the queries; the others have the keys
};

// Adjoint on 16-byte pieces. A CTA has query heads or key heads, so that it
// holds one weight and one sum; both kinds walk their units in grid order.
constexpr int BWD_UNIT = 4;
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 2) k_qk_bwd(const __grid_constant__ BwdArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, HPW = 32 / LPH;
    __shared__ float sum[WARPS][MAX_HD];
    tc::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPH, li = lane % LPH, e0 = li * V;
    const bool in = e0 < a.hd, isq = (int)blockIdx.x < a.q_ctas;
    const int heads = isq ? a.h : a.hkv, per = isq ? a.per[0] : a.per[1], units = isq ? a.units[0] : a.units[1];
    const i64 xs = isq ? a.q_stride : a.k_stride, gs = isq ? a.gq_stride : a.gk_stride;
    const T* const xp = (const T*)(isq ? a.q : a.k) + e0;
    const T* const gp = (const T*)(isq ? a.gq : a.gk) + e0;
    T* const dp = (T*)(isq ? a.dq : a.dk) + e0;
    float w[V], acc[V];
#pragma unroll
    for (int u = 0; u < V; ++u) w[u] = acc[u] = 0.f;
    if (in) ldv<float, V>((isq ? a.wq : a.wk) + e0, w);
    const i64 all = a.tokens * units;
    const int cta = isq ? blockIdx.x : blockIdx.x - a.q_ctas, ctas = isq ? a.q_ctas : gridDim.x - a.q_ctas;
    for (i64 unit = (i64)cta * WARPS + warp; unit < all; unit += (i64)ctas * WARPS) {
        const i64 tok = units == 1 ? unit : unit / units;
        const int head0 = (int)(unit - tok * units) * per * HPW + sub;
        uint4 xr[BWD_UNIT], yr[BWD_UNIT];
#pragma unroll
        for (int g = 0; g < BWD_UNIT; ++g) {
            const int head = head0 + g * HPW;
            xr[g] = yr[g] = make_uint4(0, 0, 0, 0);
            if (g < per && in && head < heads) {
                xr[g] = *(const uint4*)(xp + tok * xs + (i64)head * a.hd);
                yr[g] = *(const uint4*)(gp + tok * gs + (i64)head * a.hd);
            }
        }
        const int p = a.pos ? a.pos[tok] : (int)(tok % a.s);
        float2 cs[V / 2];
        if (in)
#pragma unroll
            for (int u = 0; u < V / 2; ++u) {
                cs[u] = cos_sin<T>(p, f.turn[li * (V / 2) + u]);
                cs[u].y = -cs[u].y;
            }
#pragma unroll
        for (int g = 0; g < BWD_UNIT; ++g) {
            if (g >= per) break;
            const int head = head0 + g * HPW;
            const bool on = in && head < heads;
            float x[V], y[V];
            unpack<T, V>(xr[g], x);
            unpack<T, V>(yr[g], y);
            if (on) rotate<V>(y, cs);
            float ss = 0.f, dot = 0.f;
#pragma unroll
            for (int u = 0; u < V; ++u) {
                ss = fmaf(x[u], x[u], ss);
                dot = fmaf(y[u] * w[u], x[u], dot);
            }
            const float r = rsqrtf(group_sum<LPH>(ss) / (float)a.hd + a.eps);
            dot = group_sum<LPH>(dot) * r / (float)a.hd;
            if (!on) continue;
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const float xh = x[u] * r;
                acc[u] = fmaf(y[u], xh, acc[u]);
                x[u] = r * (y[u] * w[u] - xh * dot);
            }
            stv<T, V>(dp + (tok * heads + head) * a.hd, x);
        }
    }
    // the groups of a warp, then the warps of the CTA, each in a fixed order
#pragma unroll
    for (int u = 0; u < V; ++u) {
#pragma unroll
        for (int o = 16; o >= LPH; o >>= 1) acc[u] += __shfl_xor_sync(0xffffffffu, acc[u], o);
        if (sub == 0 && in) sum[warp][e0 + u] = acc[u];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.hd; e += WARPS * 32) {
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < WARPS; ++j) v += sum[j][e];
        a.part[(i64)blockIdx.x * a.hd + e] = v;
    }
}

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) k_qk_bwd_any(const __grid_constant__ BwdArgs a, const __grid_constant__ Freq f) {
    __shared__ float sum[WARPS][2][MAX_HD];
    tc::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = a.h + a.hkv;
    float acc[2][2 * PAIRS];
#pragma unroll
    for (int u = 0; u < 2 * PAIRS; ++u) acc[0][u] = acc[1][u] = 0.f;
    for (i64 row = (i64)blockIdx.x * WARPS + warp; row < a.tokens * heads; row += (i64)gridDim.x * WARPS) {
        const i64 tok = row / heads;
        const int head = (int)(row - tok * heads);
        const bool isq = head < a.h;
        const int hk = head - a.h;
        const T* x = isq ? (const T*)a.q + tok * a.q_stride + (i64)head * a.hd
                         : (const T*)a.k + tok * a.k_stride + (i64)hk * a.hd;
        const T* gy = isq ? (const T*)a.gq + tok * a.gq_stride + (i64)head * a.hd
                          : (const T*)a.gk + tok * a.gk_stride + (i64)hk * a.hd;
        T* d = isq ? (T*)a.dq + (tok * a.h + head) * a.hd : (T*)a.dk + (tok * a.hkv + hk) * a.hd;
        const float* w = isq ? a.wq : a.wk;
        const int p = a.pos ? a.pos[tok] : (int)(tok % a.s);
        float v[2 * PAIRS], g[2 * PAIRS], ss = 0.f, dot = 0.f;
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) {
            const int i = lane + 32 * u;
            v[2 * u] = v[2 * u + 1] = g[2 * u] = g[2 * u + 1] = 0.f;
            if (i < a.hd / 2) {
                v[2 * u] = ld(x + 2 * i);
                v[2 * u + 1] = ld(x + 2 * i + 1);
                const float2 cs = cos_sin<T>(p, f.turn[i]);
                const float y0 = ld(gy + 2 * i), y1 = ld(gy + 2 * i + 1);
                g[2 * u] = y0 * cs.x + y1 * cs.y;
                g[2 * u + 1] = y1 * cs.x - y0 * cs.y;
                dot = fmaf(g[2 * u] * w[2 * i], v[2 * u], fmaf(g[2 * u + 1] * w[2 * i + 1], v[2 * u + 1], dot));
            }
            ss = fmaf(v[2 * u], v[2 * u], fmaf(v[2 * u + 1], v[2 * u + 1], ss));
        }
        const float r = rsqrtf(warp_sum(ss) / (float)a.hd + a.eps);
        dot = warp_sum(dot) * r / (float)a.hd;
#pragma unroll
        for (int u = 0; u < 2 * PAIRS; ++u) {
            const int e = 2 * (lane + 32 * (u / 2)) + (u & 1);
            if (e >= a.hd) continue;
            const float xh = v[u] * r;
            acc[0][u] += isq ? g[u] * xh : 0.f;
            acc[1][u] += isq ? 0.f : g[u] * xh;
            st(d + e, r * (g[u] * w[e] - xh * dot));
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int u = 0; u < 2 * PAIRS; ++u) {
            const int e = 2 * (lane + 32 * (u / 2)) + (u & 1);
            if (e < a.hd) sum[warp][m][e] = acc[m][u];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.hd; i += WARPS * 32) {
        const int m = i >= a.hd, e = i - m * a.hd;
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < WARPS; ++j) v += sum[j][m][e];
        a.part[((i64)m * gridDim.x + blockIdx.x) * a.hd + e] = v;
    }
}

// dw = the CTAs' sums added up in a fixed order: 8 columns a CTA, 32 row
// groups of which each adds every 32nd row, then the groups in order.
// Columns [0, hd) are wq's, over rows [0, rows_q); the rest wk's, over the
// rows_k rows behind them.
constexpr int FIN_COLS = 8, FIN_ROWS = 32;
__global__ void __launch_bounds__(FIN_COLS * FIN_ROWS) k_qk_dw(const float* __restrict__ part, int rows_q, int rows_k, int hd,
                                                              float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float s[FIN_ROWS][FIN_COLS];
    const int cx = threadIdx.x % FIN_COLS, ry = threadIdx.x / FIN_COLS, col = blockIdx.x * FIN_COLS + cx;
    const bool isq = col < hd;
    const int e = isq ? col : col - hd, r0 = isq ? 0 : rows_q, rows = isq ? rows_q : rows_k;
    tc::grid_dependency_wait();
    float v = 0.f;
    if (col < 2 * hd)
#pragma unroll 8
        for (int r = ry; r < rows; r += FIN_ROWS) v += __ldcg(part + (i64)(r0 + r) * hd + e);
    s[ry][cx] = v;
    __syncthreads();
    if (ry == 0 && col < 2 * hd) {
        v = 0.f;
#pragma unroll
        for (int r = 0; r < FIN_ROWS; ++r) v += s[r][cx];
        (isq ? dwq : dwk)[e] = v;
    }
}

// ------------------------------------------------------------ append
struct AppendArgs {
    const void *q, *k, *v;  // q may be null (then h = 0)
    i64 q_stride, k_stride, v_stride;
    const float *wq, *wk;  // null: no norm
    void *qo, *kc, *vc;    // caches [pages, hkv, page, hd]
    const int32_t *table, *lens, *cu;  // cu null: token t is the one new token of sequence t
    i64 tokens, seqs;
    int h, hkv, hd, page, max_pages;
    i64 pages;
    float eps;
    int per, units;
    int* err;
};

// The cache row of (seq, pos), kv head 0, or -1 (and *err set) where there is none.
__device__ __forceinline__ i64 cache_row(const AppendArgs& a, i64 seq, int pos) {
    const i64 at = place::cache_index(a.table, seq, pos, a.page, a.max_pages, a.pages, a.hkv, a.hd);
    if (at < 0 && a.err) atomicExch(a.err, 1);
    return at;
}

// Rows of a token: H query heads to qo, Hkv key heads and Hkv value heads to
// their slot. Query rows of a token that belongs to no sequence become zero.
// The rows are on their way before the token's place is looked up.
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 3) k_append(const __grid_constant__ AppendArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, HPW = 32 / LPH;
    const int lane = threadIdx.x & 31, sub = lane / LPH, li = lane % LPH, e0 = li * V, rows = a.h + 2 * a.hkv;
    const bool in = e0 < a.hd, norm = a.wq != nullptr;
    float wq[V], wk[V];
#pragma unroll
    for (int u = 0; u < V; ++u) wq[u] = wk[u] = 1.f;
    if (in && norm) {
        ldv<float, V>(a.wq + e0, wq);
        ldv<float, V>(a.wk + e0, wk);
    }
    const i64 all = a.tokens * a.units;
    for (i64 unit = (i64)blockIdx.x * WARPS + (threadIdx.x >> 5); unit < all; unit += (i64)gridDim.x * WARPS) {
        const i64 tok = a.units == 1 ? unit : unit / a.units;
        const int row0 = (int)(unit - tok * a.units) * a.per * HPW + sub;
        const T* qrow = (const T*)a.q + tok * a.q_stride + e0;
        const T* krow = (const T*)a.k + tok * a.k_stride + e0;
        const T* vrow = (const T*)a.v + tok * a.v_stride + e0;
        uint4 raw[UNIT];
#pragma unroll
        for (int g = 0; g < UNIT; ++g) {
            const int row = row0 + g * HPW, kr = row - a.h, vr = kr - a.hkv;
            raw[g] = make_uint4(0, 0, 0, 0);
            if (g < a.per && in && row < rows)
                raw[g] = *(const uint4*)(kr < 0 ? qrow + (i64)row * a.hd : vr < 0 ? krow + (i64)kr * a.hd : vrow + (i64)vr * a.hd);
        }
        i64 seq = 0;
        const int p = place::token_position(a.lens, a.cu, a.seqs, tok, seq);
        const i64 base = p >= 0 ? cache_row(a, seq, p) : -1;
        float2 cs[V / 2];
        if (in)
#pragma unroll
            for (int u = 0; u < V / 2; ++u) cs[u] = cos_sin<T>(p, f.turn[li * (V / 2) + u]);
        T* qo = (T*)a.qo + tok * a.h * a.hd + e0;
#pragma unroll
        for (int g = 0; g < UNIT; ++g) {
            if (g >= a.per) break;
            const int row = row0 + g * HPW, kr = row - a.h, vr = kr - a.hkv;
            const bool on = in && row < rows;
            float r = 1.f, x[V];
            unpack<T, V>(raw[g], x);
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int u = 0; u < V; ++u) ss = fmaf(x[u], x[u], ss);
                r = rsqrtf(group_sum<LPH>(ss) / (float)a.hd + a.eps);
            }
            if (!on) continue;
            if (vr < 0) {
#pragma unroll
                for (int u = 0; u < V; ++u) x[u] = p >= 0 ? x[u] * r * (kr < 0 ? wq[u] : wk[u]) : 0.f;
                rotate<V>(x, cs);
            }
            if (kr < 0) stv<T, V>(qo + (i64)row * a.hd, x);
            else if (base >= 0) stv<T, V>((T*)(vr < 0 ? a.kc : a.vc) + base + (i64)(vr < 0 ? kr : vr) * a.page * a.hd + e0, x);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) k_append_any(const __grid_constant__ AppendArgs a, const __grid_constant__ Freq f) {
    const int lane = threadIdx.x & 31, rows = a.h + 2 * a.hkv;
    const i64 unit = (i64)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const i64 tok = unit / rows;
    if (tok >= a.tokens) return;
    const int row = (int)(unit - tok * rows);
    const int kind = row < a.h ? 0 : row < a.h + a.hkv ? 1 : 2, head = kind == 0 ? row : kind == 1 ? row - a.h : row - a.h - a.hkv;
    i64 seq = 0;
    const int p = place::token_position(a.lens, a.cu, a.seqs, tok, seq);
    const i64 base = p >= 0 ? cache_row(a, seq, p) : -1;
    if (kind != 0 && base < 0) return;
    const T* x = kind == 0 ? (const T*)a.q + tok * a.q_stride : kind == 1 ? (const T*)a.k + tok * a.k_stride : (const T*)a.v + tok * a.v_stride;
    x += (i64)head * a.hd;
    T* y = kind == 0 ? (T*)a.qo + (tok * a.h + head) * a.hd : (T*)(kind == 1 ? a.kc : a.vc) + base + (i64)head * a.page * a.hd;
    float v[2 * PAIRS], ss = 0.f;
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        const int i = lane + 32 * u;
        v[2 * u] = v[2 * u + 1] = 0.f;
        if (i < a.hd / 2 && p >= 0) {
            v[2 * u] = ld(x + 2 * i);
            v[2 * u + 1] = ld(x + 2 * i + 1);
        }
        ss = fmaf(v[2 * u], v[2 * u], fmaf(v[2 * u + 1], v[2 * u + 1], ss));
    }
    const float* w = kind == 2 ? nullptr : kind == 0 ? a.wq : a.wk;
    const float r = w ? rsqrtf(warp_sum(ss) / (float)a.hd + a.eps) : 1.f;
#pragma unroll
    for (int u = 0; u < PAIRS; ++u) {
        const int i = lane + 32 * u;
        if (i >= a.hd / 2) continue;
        float x0 = v[2 * u], x1 = v[2 * u + 1];
        if (w) {
            x0 = x0 * r * w[2 * i];
            x1 = x1 * r * w[2 * i + 1];
        }
        if (kind < 2 && p >= 0) {
            const float2 cs = cos_sin<T>(p, f.turn[i]);
            const float t = x0 * cs.x - x1 * cs.y;
            x1 = x0 * cs.y + x1 * cs.x;
            x0 = t;
        }
        st(y + 2 * i, x0);
        st(y + 2 * i + 1, x1);
    }
}

// ------------------------------------------------------------ launchers
// Groups of HPW rows that a unit takes of one token: as many as fit (the
// sines are then taken once a token), unless that would leave SMs without warps.
static int groups_per_unit(Context* c, i64 tokens, int groups, int most) {
    const i64 want = (i64)c->sm_count * 16;
    const int units = cdiv(groups, (int)std::max<i64>(1, std::min<i64>(most, tokens * groups / want)));
    return cdiv(groups, units);
}

static int lanes_of(int hd, int vec) {
    int l = 4;
    while (l * vec < hd) l <<= 1;
    return l;
}

static void check_heads(i64 tokens, i64 h, i64 hkv, i64 hd, const char* what) {
    CATNN_CHECK(hd >= 2 && hd % 2 == 0 && hd <= MAX_HD, CATNN_ERR_UNSUPPORTED,
                std::string(what) + ": head_dim must be even and at most 256");
    CATNN_CHECK(tokens >= 0 && h >= 0 && hkv >= 1 && h + 2 * hkv <= 65536 && tokens <= (1ll << 31) - 1, CATNN_ERR_SHAPE,
                std::string(what) + ": sizes");
}
static int grid_of(i64 warps, const char* what) {
    const i64 g = (warps + WARPS - 1) / WARPS;
    CATNN_CHECK(g <= 0x7fffffff, CATNN_ERR_SHAPE, std::string(what) + ": too many rows for one call");
    return (int)g;
}

static bool rows_ok(const void* p, i64 stride, i64 hd, int vec) {
    return hd % vec == 0 && stride % vec == 0 && aligned_to(p, 16);
}

#define BY_LANES(L, F, T)                     \
    switch (L) {                              \
        case 4: F(T, 4); break;               \
        case 8: F(T, 8); break;               \
        case 16: F(T, 16); break;             \
        default: F(T, 32); break;             \
    }

}  // namespace qkn

using namespace qkn;

void qk_norm_rope_fwd(Context* c, const void* q, i64 q_stride, const void* k, i64 k_stride, const float* wq, const float* wk,
                      const int32_t* pos, void* qo, void* ko, i64 b, i64 s, i64 h, i64 hkv, i64 hd, double theta, float eps,
                      int dtype) {
    const i64 tokens = b * s;
    check_heads(tokens, h, hkv, hd, "qk_norm_rope");
    if (tokens == 0) return;
    const Freq& f = freq_of(c, hd, theta);
    FwdArgs a{q, k, q_stride, k_stride, wq, wk, pos, qo, ko, tokens, s, (int)h, (int)hkv, (int)hd, eps, 1, 1};
    const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
    if (lph <= 32 && rows_ok(q, q_stride, hd, vec) && rows_ok(k, k_stride, hd, vec) && aligned_to(qo, 16) &&
        aligned_to(ko, 16) && aligned_to(wq, 16) && aligned_to(wk, 16)) {
        const int groups = cdiv(h + hkv, 32 / lph);
        a.per = groups_per_unit(c, tokens, groups, UNIT);
        a.units = cdiv(groups, a.per);
        const int grid = (int)std::min<i64>((tokens * a.units + WARPS - 1) / WARPS, c->sm_count * 3);
#define RUN(T, L) k_qk_fwd<T, L><<<grid, WARPS * 32, 0, c->stream>>>(a, f)
        if (dtype == CATNN_BF16) { BY_LANES(lph, RUN, bf16) } else { BY_LANES(lph, RUN, float) }
#undef RUN
    } else {
        const int grid = grid_of(tokens * (h + hkv), "qk_norm_rope");
        if (dtype == CATNN_BF16) k_qk_fwd_any<bf16><<<grid, WARPS * 32, 0, c->stream>>>(a, f);
        else k_qk_fwd_any<float><<<grid, WARPS * 32, 0, c->stream>>>(a, f);
    }
    launched(c);
}

// CTAs of the adjoint: what the SMs hold at once, each walking many tokens,
// because every CTA adds a row to the weight sums.
static i64 qk_bwd_ctas(Context* c, i64 rows) { return std::min<i64>((i64)c->sm_count * 2, (rows + WARPS - 1) / WARPS); }

// At least one CTA each for queries and keys, two rows a CTA where it has both.
size_t qk_norm_rope_bwd_workspace(Context* c, i64 b, i64 s, i64 h, i64 hkv, i64 hd) {
    return (size_t)(qk_bwd_ctas(c, b * s * (h + hkv)) + 1) * 2 * hd * sizeof(float);
}

void qk_norm_rope_bwd(Context* c, const void* q, i64 q_stride, const void* k, i64 k_stride, const float* wq, const float* wk,
                      const int32_t* pos, const void* gq, i64 gq_stride, const void* gk, i64 gk_stride, void* dq, void* dk,
                      float* dwq, float* dwk, i64 b, i64 s, i64 h, i64 hkv, i64 hd, double theta, float eps, int dtype,
                      float* work) {
    const i64 tokens = b * s;
    check_heads(tokens, h, hkv, hd, "qk_norm_rope backward");
    const Freq& f = freq_of(c, hd, theta);
    BwdArgs a{q, k, gq, gk, q_stride, k_stride, gq_stride, gk_stride, wq, wk, pos, dq, dk, work, tokens, s, (int)h, (int)hkv,
              (int)hd, eps, {1, 1}, {1, 1}, 0};
    int rows_q = 0, rows_k = 0;
    if (tokens > 0) {
        const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
        if (lph <= 32 && rows_ok(q, q_stride, hd, vec) && rows_ok(k, k_stride, hd, vec) && rows_ok(gq, gq_stride, hd, vec) &&
            rows_ok(gk, gk_stride, hd, vec) && aligned_to(dq, 16) && aligned_to(dk, 16) && aligned_to(wq, 16) &&
            aligned_to(wk, 16)) {
            const int groups[2] = {cdiv(h, 32 / lph), cdiv(hkv, 32 / lph)};
            for (int m = 0; m < 2; ++m) {
                a.per[m] = groups_per_unit(c, tokens, groups[m], BWD_UNIT);
                a.units[m] = cdiv(groups[m], a.per[m]);
            }
            // CTAs in the proportion of the row groups, none without a unit
            const i64 uq = tokens * a.units[0], uk = tokens * a.units[1], ctas = std::max<i64>(2, qk_bwd_ctas(c, uq + uk));
            const i64 share = ctas * groups[0] / (groups[0] + groups[1]);
            rows_q = (int)std::min<i64>(std::max<i64>(1, std::min(share, ctas - 1)), (uq + WARPS - 1) / WARPS);
            rows_k = (int)std::min<i64>(ctas - rows_q, (uk + WARPS - 1) / WARPS);
            a.q_ctas = rows_q;
#define RUN(T, L) k_qk_bwd<T, L><<<rows_q + rows_k, WARPS * 32, 0, c->stream>>>(a, f)
            if (dtype == CATNN_BF16) { BY_LANES(lph, RUN, bf16) } else { BY_LANES(lph, RUN, float) }
#undef RUN
        } else {
            rows_q = rows_k = (int)qk_bwd_ctas(c, tokens * (h + hkv));
            if (dtype == CATNN_BF16) k_qk_bwd_any<bf16><<<rows_q, WARPS * 32, 0, c->stream>>>(a, f);
            else k_qk_bwd_any<float><<<rows_q, WARPS * 32, 0, c->stream>>>(a, f);
        }
        launched(c);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cdiv(2 * hd, FIN_COLS));
    cfg.blockDim = dim3(FIN_COLS * FIN_ROWS);
    cfg.stream = c->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = tokens > 0 ? 1 : 0;  // with no tokens there is no first kernel that lets this one start
    CUDA_OK(cudaLaunchKernelEx(&cfg, k_qk_dw, (const float*)work, rows_q, rows_k, (int)hd, dwq, dwk));
    launched(c);
}

void kv_append(Context* c, const void* q, i64 q_stride, const void* k, i64 k_stride, const void* v, i64 v_stride,
               const float* wq, const float* wk, void* qo, void* kc, void* vc, const int32_t* table, const int32_t* lens,
               const int32_t* cu, i64 tokens, i64 seqs, i64 h, i64 hkv, i64 hd, i64 pages, i64 page, i64 max_pages,
               double theta, float eps, int dtype, int* err) {
    check_heads(tokens, h, hkv, hd, "kv_append");
    if (tokens == 0) return;
    const Freq& f = freq_of(c, hd, theta);
    AppendArgs a{q, k, v, q_stride, k_stride, v_stride, wq, wk, qo, kc, vc, table, lens, cu, tokens, seqs, (int)h, (int)hkv,
                 (int)hd, (int)page, (int)max_pages, pages, eps, 1, 1, err};
    const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
    if (lph <= 32 && (!q || rows_ok(q, q_stride, hd, vec)) && rows_ok(k, k_stride, hd, vec) && rows_ok(v, v_stride, hd, vec) &&
        aligned_to(qo, 16) && aligned_to(kc, 16) && aligned_to(vc, 16) && aligned_to(wq, 16) && aligned_to(wk, 16)) {
        const int groups = cdiv(h + 2 * hkv, 32 / lph);
        a.per = groups_per_unit(c, tokens, groups, UNIT);
        a.units = cdiv(groups, a.per);
        const int grid = (int)std::min<i64>((tokens * a.units + WARPS - 1) / WARPS, c->sm_count * 3);
#define RUN(T, L) k_append<T, L><<<grid, WARPS * 32, 0, c->stream>>>(a, f)
        if (dtype == CATNN_BF16) { BY_LANES(lph, RUN, bf16) } else { BY_LANES(lph, RUN, float) }
#undef RUN
    } else {
        const int grid = grid_of(tokens * (h + 2 * hkv), "kv_append");
        if (dtype == CATNN_BF16) k_append_any<bf16><<<grid, WARPS * 32, 0, c->stream>>>(a, f);
        else k_append_any<float><<<grid, WARPS * 32, 0, c->stream>>>(a, f);
    }
    launched(c);
}

}  // namespace catnn
