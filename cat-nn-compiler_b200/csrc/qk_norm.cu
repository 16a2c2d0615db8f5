// RMS norm of every query and key head with the position rotation in the
// same pass (forward and adjoint), and the append of new keys and values to
// a paged cache with both applied on the way.
//
// With x one head's row of hd values, r = (mean(x²) + eps)^(-1/2) and R(p)
// the rotation of the pairs (2i, 2i+1) by p·θ^(-2i/hd):
//   forward  y = R(p)·(x·r·w)
//   adjoint  g = R(p)ᵀ·dy, x̂ = x·r, dw = Σ_rows g·x̂,
//            dx = r·(g·w − x̂·mean(g·w·x̂))
// Every kernel reads its rows once and writes them once, so HBM bounds them;
// what holds them off its rate is latency at low occupancy: a warp asks for a
// batch of rows, computes, stores, and only then asks for the next, and the
// registers of a batch leave 16 to 24 warps an SM. (Instruction issue does not:
// at four a cycle and SM it would take 9, 14 and 19 us of the times below.)
// Measured, bf16: 16384 tokens of 16 + 4 heads of 64 forward 17.1 us (4.9 TB/s,
// 0.75 of the copy rate), adjoint 27.3 us (4.6 TB/s); append of 14087 tokens of
// 16 + 2 x 4 heads of 128 with the norm 39.7 us (4.1 TB/s); one token 2.7 us, an
// append of 32 single ones 4.4.
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
#include "row_deal.cuh"
#include "tc_prims.cuh"

namespace catnn {
namespace qkn {

using namespace deal;

constexpr int MAX_HD = 256;

// θ^(-2i/hd) / 2π: the pair's turns per position, in f64 because a far
// position times a rounded f32 frequency is off by more than any rounding
// (up to 0.06 radians at position 10^6).
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
// below the 2^-8 of the rounding that follows.
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

// Two floats in one register pair, for the instructions that work on both.
// They shorten what a warp does between its loads (54 -> 30 us in the adjoint):
// a lane's values are taken two pairs at a time: X0 = the first elements of
// pairs i and i + 1, X1 = their second elements.
using namespace tc::pairs;

// Read once: first to leave the L2 (adjoint 28.5 -> 27.3 us at 16384 tokens of 16 + 4 heads of 64).
__device__ __forceinline__ uint4 ld16(const void* p) { return __ldcs((const uint4*)p); }
__device__ __forceinline__ void st16(void* p, const uint4& v) { *(uint4*)p = v; }

// 16 bytes as packed pairs, and back.
template <typename T> constexpr int NP = VEC<T> / 4;
template <typename T> __device__ __forceinline__ void unpack(const uint4& r, f2 (&x0)[NP<T>], f2 (&x1)[NP<T>]) {
    if constexpr (sizeof(T) == 4) {
        x0[0] = pack2(__uint_as_float(r.x), __uint_as_float(r.z));
        x1[0] = pack2(__uint_as_float(r.y), __uint_as_float(r.w));
    } else {
        x0[0] = pack2(__uint_as_float(r.x << 16), __uint_as_float(r.y << 16));
        x1[0] = pack2(__uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y & 0xffff0000u));
        x0[1] = pack2(__uint_as_float(r.z << 16), __uint_as_float(r.w << 16));
        x1[1] = pack2(__uint_as_float(r.z & 0xffff0000u), __uint_as_float(r.w & 0xffff0000u));
    }
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t*)&h;
}
template <typename T> __device__ __forceinline__ uint4 repack(const f2 (&x0)[NP<T>], const f2 (&x1)[NP<T>]) {
    const float2 a = split2(x0[0]), b = split2(x1[0]);
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(a.x), __float_as_uint(b.x), __float_as_uint(a.y), __float_as_uint(b.y));
    } else {
        const float2 c = split2(x0[1]), d = split2(x1[1]);
        return make_uint4(bf16x2(a.x, b.x), bf16x2(a.y, b.y), bf16x2(c.x, d.x), bf16x2(c.y, d.y));
    }
}

// A lane's cosines and sines at a position.
template <typename T> struct Turn {
    f2 c[NP<T>], s[NP<T>];
    __device__ __forceinline__ void at(int pos, const Freq& f, int pair0) {
#pragma unroll
        for (int j = 0; j < NP<T>; ++j) {
            const float2 a = cos_sin<T>(pos, f.turn[pair0 + 2 * j]), b = cos_sin<T>(pos, f.turn[pair0 + 2 * j + 1]);
            c[j] = pack2(a.x, b.x);
            s[j] = pack2(a.y, b.y);
        }
    }
};
// The norm's weights of a lane's pairs, out of shared memory.
template <typename T> __device__ __forceinline__ void weights(const float* w, f2 (&w0)[NP<T>], f2 (&w1)[NP<T>]) {
#pragma unroll
    for (int j = 0; j < NP<T>; ++j) {
        const float4 v = *(const float4*)(w + 4 * j);
        w0[j] = pack2(v.x, v.z);
        w1[j] = pack2(v.y, v.w);
    }
}
// Weight and rotation in one: y0 = x0·a + x1·b, y1 = x0·c + x1·d.
template <typename T> struct Coef {
    f2 a[NP<T>], b[NP<T>], c[NP<T>], d[NP<T>];
    __device__ __forceinline__ void of(const Turn<T>& t, const float* w) {
        f2 w0[NP<T>], w1[NP<T>];
        weights<T>(w, w0, w1);
        const f2 minus = pack2(-1.f, -1.f);
#pragma unroll
        for (int j = 0; j < NP<T>; ++j) {
            a[j] = mul2(w0[j], t.c[j]);
            b[j] = mul2(mul2(w1[j], t.s[j]), minus);
            c[j] = mul2(w0[j], t.s[j]);
            d[j] = mul2(w1[j], t.c[j]);
        }
    }
};

// One row: its norm (where `norm`), weights and rotation.
template <typename T, int LPH>
__device__ __forceinline__ uint4 norm_turn(const uint4& raw, const Coef<T>& k, bool norm, float inv_hd, float eps) {
    f2 x0[NP<T>], x1[NP<T>], y0[NP<T>], y1[NP<T>];
    unpack<T>(raw, x0, x1);
    f2 r = pack2(1.f, 1.f);
    if (norm) {
        f2 ss = mul2(x0[0], x0[0]);
        ss = fma2(x1[0], x1[0], ss);
        if (NP<T> > 1) {
            ss = fma2(x0[NP<T> - 1], x0[NP<T> - 1], ss);
            ss = fma2(x1[NP<T> - 1], x1[NP<T> - 1], ss);
        }
        const float v = rsqrtf(fmaf(group_sum<LPH>(sum2(ss)), inv_hd, eps));
        r = pack2(v, v);
    }
#pragma unroll
    for (int j = 0; j < NP<T>; ++j) {
        y0[j] = mul2(fma2(x1[j], k.b[j], mul2(x0[j], k.a[j])), r);
        y1[j] = mul2(fma2(x1[j], k.d[j], mul2(x0[j], k.c[j])), r);
    }
    return repack<T>(y0, y1);
}

// The weights in shared memory, once a CTA; 1 where there are none.
__device__ __forceinline__ void load_weights(float (&sw)[2][MAX_HD], const float* wq, const float* wk, int hd) {
    for (int i = threadIdx.x; i < MAX_HD; i += blockDim.x) {
        sw[0][i] = i < hd && wq ? wq[i] : 1.f;
        sw[1][i] = i < hd && wk ? wk[i] : 1.f;
    }
    __syncthreads();
}

// A warp's share of the rows (row_deal.cuh).
__device__ __forceinline__ Share my_share(const Deal& d) { return share_of(d, blockIdx.x * WARPS + (threadIdx.x >> 5)); }

struct FwdArgs {
    const void *q, *k;
    i64 q_stride, k_stride;  // elements between tokens
    const float *wq, *wk;
    const int32_t* pos;  // [tokens], or null: token % s
    void *qo, *ko;
    i64 tokens, s;
    int h, hkv, hd;
    float eps, inv_hd;
    Deal deal;
    int gq;  // row groups of a token: gq of its query heads, then those of its key heads
};

// Forward on 16-byte pieces. A group is the HPW = 32 / LPH heads that a warp
// takes at once. A warp walks its tokens, and each one's groups a batch at a
// time; a batch's rows are all on their way before the token's sines are taken.
constexpr int BATCH = 6;
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 3) k_qk_fwd(const __grid_constant__ FwdArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, HPW = 32 / LPH;
    __shared__ __align__(16) float sw[2][MAX_HD];
    const int lane = threadIdx.x & 31, sub = lane / LPH, e0 = lane % LPH * V, step = HPW * a.hd, off = sub * a.hd + e0;
    const bool in = e0 < a.hd;
    load_weights(sw, a.wq, a.wk, a.hd);
    const Share w = my_share(a.deal);
    for (int tok = w.t0; tok < w.t1; tok += w.dt) {
        Turn<T> t;
        for (int g0 = w.g0; g0 < w.g1; g0 += BATCH) {
            const int nq = a.gq - g0, n = w.g1 - g0;  // group g is a query group for g < nq
            const T* const q = (const T*)a.q + tok * a.q_stride + off + g0 * step;
            const T* const k = (const T*)a.k + tok * a.k_stride + off - nq * step;
            const int hq = in ? a.h - g0 * HPW - sub : 0, hk = in ? a.hkv + nq * HPW - sub : 0;  // group g is there for g·HPW below
            uint4 raw[BATCH];
#pragma unroll
            for (int g = 0; g < BATCH; ++g) {
                raw[g] = make_uint4(0, 0, 0, 0);
                if (g < n && g * HPW < (g < nq ? hq : hk)) raw[g] = ld16((g < nq ? q : k) + g * step);
            }
            if (g0 == w.g0) t.at(a.pos ? a.pos[tok] : (int)((unsigned)tok % (unsigned)a.s), f, e0 / 2);
            T* const qo = (T*)a.qo + (i64)tok * a.h * a.hd + off + g0 * step;
            T* const ko = (T*)a.ko + (i64)tok * a.hkv * a.hd + off - nq * step;
            Coef<T> c;
            if (nq > 0) c.of(t, sw[0] + e0);
#pragma unroll
            for (int g = 0; g < BATCH; ++g) {
                if (g >= n) break;
                if (g == max(nq, 0)) c.of(t, sw[1] + e0);
                const uint4 y = norm_turn<T, LPH>(raw[g], c, true, a.inv_hd, a.eps);
                if (g * HPW < (g < nq ? hq : hk)) st16((g < nq ? qo : ko) + g * step, y);
            }
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
    float* part;  // [2][CTAs][hd]: each CTA's sums for wq, then for wk
    i64 tokens, s;
    int h, hkv, hd;
    float eps, inv_hd;
    Deal deal;
    int groups_q;  // as in the forward
};

// Adjoint on 16-byte pieces, dealt out as the forward; both weight sums stay
// in registers over all of a warp's rows.
constexpr int BWD_BATCH = 5;
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 2) k_qk_bwd(const __grid_constant__ BwdArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, N = NP<T>, HPW = 32 / LPH;
    __shared__ __align__(16) float sw[2][MAX_HD];
    __shared__ float sum[WARPS][MAX_HD];
    tc::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPH, e0 = lane % LPH * V, step = HPW * a.hd;
    const int off = sub * a.hd + e0;
    const bool in = e0 < a.hd;
    load_weights(sw, a.wq, a.wk, a.hd);
    f2 acc[2][2][N];  // of queries and keys, of first and second elements
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[m][0][j] = acc[m][1][j] = pack2(0.f, 0.f);
    const f2 minus = pack2(-1.f, -1.f);
    const Share w = my_share(a.deal);
    for (int tok = w.t0; tok < w.t1; tok += w.dt) {
      Turn<T> t;
      f2 ns[N];
      for (int b0 = w.g0; b0 < w.g1; b0 += BWD_BATCH) {
        const int nq = a.groups_q - b0, n = w.g1 - b0;
        const T* const q = (const T*)a.q + tok * a.q_stride + off + b0 * step;
        const T* const k = (const T*)a.k + tok * a.k_stride + off - nq * step;
        const T* const gq = (const T*)a.gq + tok * a.gq_stride + off + b0 * step;
        const T* const gk = (const T*)a.gk + tok * a.gk_stride + off - nq * step;
        const int hq = in ? a.h - b0 * HPW - sub : 0, hk = in ? a.hkv + nq * HPW - sub : 0;
        uint4 xr[BWD_BATCH], yr[BWD_BATCH];
#pragma unroll
        for (int g = 0; g < BWD_BATCH; ++g) {
            xr[g] = yr[g] = make_uint4(0, 0, 0, 0);
            if (g < n && g * HPW < (g < nq ? hq : hk)) {
                xr[g] = ld16((g < nq ? q : k) + g * step);
                yr[g] = ld16((g < nq ? gq : gk) + g * step);
            }
        }
        if (b0 == w.g0) {
            t.at(a.pos ? a.pos[tok] : (int)((unsigned)tok % (unsigned)a.s), f, e0 / 2);
#pragma unroll
            for (int j = 0; j < N; ++j) ns[j] = mul2(t.s[j], minus);
        }
        T* const dq = (T*)a.dq + (i64)tok * a.h * a.hd + off + b0 * step;
        T* const dk = (T*)a.dk + (i64)tok * a.hkv * a.hd + off - nq * step;
        f2 w0[N], w1[N];
        weights<T>(sw[nq > 0 ? 0 : 1] + e0, w0, w1);
#pragma unroll
        for (int g = 0; g < BWD_BATCH; ++g) {
            if (g >= n) break;
            if (g > 0 && g == nq) weights<T>(sw[1] + e0, w0, w1);
            f2 x0[N], x1[N], y0[N], y1[N], g0_[N], g1_[N];
            unpack<T>(xr[g], x0, x1);
            unpack<T>(yr[g], y0, y1);
            f2 ss = pack2(0.f, 0.f), dt = ss;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                g0_[j] = fma2(y1[j], t.s[j], mul2(y0[j], t.c[j]));  // turned back
                g1_[j] = fma2(y0[j], ns[j], mul2(y1[j], t.c[j]));
                ss = fma2(x0[j], x0[j], ss);
                ss = fma2(x1[j], x1[j], ss);
                y0[j] = mul2(g0_[j], w0[j]);
                y1[j] = mul2(g1_[j], w1[j]);
                dt = fma2(y0[j], x0[j], dt);
                dt = fma2(y1[j], x1[j], dt);
            }
            const bool on = g * HPW < (g < nq ? hq : hk);
            const float mean = fmaf(group_sum<LPH>(sum2(ss)), a.inv_hd, a.eps), r = on ? rsqrtf(mean) : 0.f;
            const float m = -(group_sum<LPH>(sum2(dt)) * r * a.inv_hd) * r;  // -r·mean(g·w·x̂)
            const f2 rr = pack2(r, r), mm = pack2(m, m);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x0[j] = mul2(x0[j], rr);
                x1[j] = mul2(x1[j], rr);
                // a row that is not there has x = 0 and r = 0 and adds nothing
                if (g < nq) {
                    acc[0][0][j] = fma2(g0_[j], x0[j], acc[0][0][j]);
                    acc[0][1][j] = fma2(g1_[j], x1[j], acc[0][1][j]);
                } else {
                    acc[1][0][j] = fma2(g0_[j], x0[j], acc[1][0][j]);
                    acc[1][1][j] = fma2(g1_[j], x1[j], acc[1][1][j]);
                }
                y0[j] = fma2(x0[j], mm, mul2(y0[j], rr));
                y1[j] = fma2(x1[j], mm, mul2(y1[j], rr));
            }
            if (on) st16((g < nq ? dq : dk) + g * step, repack<T>(y0, y1));
        }
      }
    }
    // the groups of a warp, then the warps of the CTA, each in a fixed order
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float2 v0 = split2(acc[m][0][j]), v1 = split2(acc[m][1][j]);
            float v[4] = {v0.x, v1.x, v0.y, v1.y};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int o = 16; o >= LPH; o >>= 1) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
                if (sub == 0 && in) sum[warp][e0 + 4 * j + u] = v[u];
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.hd; e += WARPS * 32) {
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) v += sum[j][e];
            a.part[((i64)m * gridDim.x + blockIdx.x) * a.hd + e] = v;
        }
        __syncthreads();
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
// Columns [0, hd) are wq's, the rest wk's, whose rows lie behind wq's.
constexpr int FIN_COLS = 8, FIN_ROWS = 32;
__global__ void __launch_bounds__(FIN_COLS * FIN_ROWS) k_qk_dw(const float* __restrict__ part, int rows, int hd,
                                                              float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float s[FIN_ROWS][FIN_COLS];
    const int cx = threadIdx.x % FIN_COLS, ry = threadIdx.x / FIN_COLS, col = blockIdx.x * FIN_COLS + cx;
    const bool isq = col < hd;
    const int e = isq ? col : col - hd, r0 = isq ? 0 : rows;
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
    float eps, inv_hd;
    Deal deal;
    int gq, gk;
    int* err;
};

// The cache row of (seq, pos), kv head 0, or -1 (and *err set) where there is none.
__device__ __forceinline__ i64 cache_row(const AppendArgs& a, int seq, int pos) {
    const i64 at = place::cache_index(a.table, seq, pos, a.page, a.max_pages, a.pages, a.hkv, a.hd);
    if (at < 0 && a.err) atomicExch(a.err, 1);
    return at;
}

// Row groups of a token: gq of its H query heads, which go to qo, then gk of
// its key heads and as many of its value heads, which go to their slots; the
// values are copied as they are. Query rows of a token that belongs to no
// sequence become zero. The rows are on their way before the token's place is
// looked up.
template <typename T, int LPH>
__global__ void __launch_bounds__(WARPS * 32, 3) k_append(const __grid_constant__ AppendArgs a, const __grid_constant__ Freq f) {
    constexpr int V = VEC<T>, HPW = 32 / LPH;
    __shared__ __align__(16) float sw[2][MAX_HD];
    const int lane = threadIdx.x & 31, sub = lane / LPH, e0 = lane % LPH * V, step = HPW * a.hd, off = sub * a.hd + e0;
    const bool in = e0 < a.hd, norm = a.wq != nullptr;
    load_weights(sw, a.wq, a.wk, a.hd);
    const Share w = my_share(a.deal);
    place::Token at;
    for (int tok = w.t0; tok < w.t1; tok += w.dt) {
        Turn<T> t;
        int p = -1;
        i64 base = -1;
        for (int g0 = w.g0; g0 < w.g1; g0 += BATCH) {
            const int nq = a.gq - g0, nk = nq + a.gk, n = w.g1 - g0;  // group g: a query group below nq, a key group below nk
            const T* const q = (const T*)a.q + tok * a.q_stride + off + g0 * step;
            const T* const k = (const T*)a.k + tok * a.k_stride + off - nq * step;
            const T* const v = (const T*)a.v + tok * a.v_stride + off - nk * step;
            const int hq = in ? a.h - g0 * HPW - sub : 0, hk = in ? a.hkv + nq * HPW - sub : 0;
            const int hv = in ? a.hkv + nk * HPW - sub : 0;
            uint4 raw[BATCH];
#pragma unroll
            for (int g = 0; g < BATCH; ++g) {
                raw[g] = make_uint4(0, 0, 0, 0);
                if (g < n && g * HPW < (g < nq ? hq : g < nk ? hk : hv))
                    raw[g] = ld16((g < nq ? q : g < nk ? k : v) + g * step);
            }
            if (g0 == w.g0) {
                at.move_to(a.lens, a.cu, (int)a.seqs, tok);
                p = at.position(tok);
                base = p >= 0 ? cache_row(a, at.seq, p) : -1;
                if (g0 < a.gq + a.gk) t.at(p, f, e0 / 2);
            }
            Coef<T> c;
            if (nq > 0) c.of(t, sw[0] + e0);
            T* const qo = (T*)a.qo + (i64)tok * a.h * a.hd + off + g0 * step;
#pragma unroll
            for (int g = 0; g < BATCH; ++g) {
                if (g >= n) break;
                if (g == max(nq, 0) && g < nk) c.of(t, sw[1] + e0);
                uint4 y = raw[g];
                if (g < nk) y = norm_turn<T, LPH>(y, c, norm, a.inv_hd, a.eps);
                if (g < nq) {
                    if (g * HPW < hq) st16(qo + g * step, p >= 0 ? y : make_uint4(0, 0, 0, 0));
                } else if (base >= 0 && g * HPW < (g < nk ? hk : hv)) {
                    const int head = (g - (g < nk ? nq : nk)) * HPW + sub;
                    st16((T*)(g < nk ? a.kc : a.vc) + base + (i64)head * a.page * a.hd + e0, y);
                }
            }
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
    int seq = 0;
    const int p = place::token_position(a.lens, a.cu, (int)a.seqs, (int)tok, seq);
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
static int lanes_of(int hd, int vec) {
    int l = 4;
    while (l * vec < hd) l <<= 1;
    return l;
}

static void check_heads(i64 tokens, i64 h, i64 hkv, i64 hd, const char* what) {
    CATNN_CHECK(hd >= 2 && hd % 2 == 0 && hd <= MAX_HD, CATNN_ERR_UNSUPPORTED,
                std::string(what) + ": head_dim must be even and at most 256");
    CATNN_CHECK(tokens >= 0 && h >= 0 && hkv >= 1 && h + 2 * hkv <= 65536 && tokens <= 0x7fff0000, CATNN_ERR_SHAPE,
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
    FwdArgs a{q, k, q_stride, k_stride, wq, wk, pos, qo, ko, tokens, s, (int)h, (int)hkv, (int)hd, eps, 1.f / (float)hd,
              {}, 0};
    const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
    if (lph <= 32 && rows_ok(q, q_stride, hd, vec) && rows_ok(k, k_stride, hd, vec) && aligned_to(qo, 16) &&
        aligned_to(ko, 16)) {
        a.gq = cdiv(h, 32 / lph);
        const int grid = deal_out(c->sm_count, tokens, a.gq + cdiv(hkv, 32 / lph), 3, false, a.deal);
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

size_t qk_norm_rope_bwd_workspace(Context* c, i64 b, i64 s, i64 h, i64 hkv, i64 hd) {
    return (size_t)adjoint_rows(c->sm_count, b * s, h + hkv) * 2 * hd * sizeof(float);
}

void qk_norm_rope_bwd(Context* c, const void* q, i64 q_stride, const void* k, i64 k_stride, const float* wq, const float* wk,
                      const int32_t* pos, const void* gq, i64 gq_stride, const void* gk, i64 gk_stride, void* dq, void* dk,
                      float* dwq, float* dwk, i64 b, i64 s, i64 h, i64 hkv, i64 hd, double theta, float eps, int dtype,
                      float* work) {
    const i64 tokens = b * s;
    check_heads(tokens, h, hkv, hd, "qk_norm_rope backward");
    const Freq& f = freq_of(c, hd, theta);
    BwdArgs a{q, k, gq, gk, q_stride, k_stride, gq_stride, gk_stride, wq, wk, pos, dq, dk, work, tokens, s, (int)h, (int)hkv,
              (int)hd, eps, 1.f / (float)hd, {}, 0};
    int ctas = 0;
    const i64 room = adjoint_rows(c->sm_count, tokens, h + hkv);  // rows of each weight sum in `work`
    const auto fits = [&] { CATNN_CHECK(ctas <= room, CATNN_ERR_INVALID, "qk_norm_rope backward: more CTAs than the workspace has rows"); };
    if (tokens > 0) {
        const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
        if (lph <= 32 && rows_ok(q, q_stride, hd, vec) && rows_ok(k, k_stride, hd, vec) && rows_ok(gq, gq_stride, hd, vec) &&
            rows_ok(gk, gk_stride, hd, vec) && aligned_to(dq, 16) && aligned_to(dk, 16)) {
            a.groups_q = cdiv(h, 32 / lph);
            ctas = deal_out(c->sm_count, tokens, a.groups_q + cdiv(hkv, 32 / lph), ADJOINT_PER_SM, false, a.deal);
            fits();
#define RUN(T, L) k_qk_bwd<T, L><<<ctas, WARPS * 32, 0, c->stream>>>(a, f)
            if (dtype == CATNN_BF16) { BY_LANES(lph, RUN, bf16) } else { BY_LANES(lph, RUN, float) }
#undef RUN
        } else {
            ctas = (int)std::min<i64>((i64)c->sm_count * ADJOINT_PER_SM, (tokens * (h + hkv) + WARPS - 1) / WARPS);
            fits();
            if (dtype == CATNN_BF16) k_qk_bwd_any<bf16><<<ctas, WARPS * 32, 0, c->stream>>>(a, f);
            else k_qk_bwd_any<float><<<ctas, WARPS * 32, 0, c->stream>>>(a, f);
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
    CUDA_OK(cudaLaunchKernelEx(&cfg, k_qk_dw, (const float*)work, ctas, (int)hd, dwq, dwk));
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
                 (int)hd, (int)page, (int)max_pages, pages, eps, 1.f / (float)hd, {}, 0, 0, err};
    const int vec = dtype == CATNN_BF16 ? 8 : 4, lph = lanes_of((int)hd, vec);
    if (lph <= 32 && (!q || rows_ok(q, q_stride, hd, vec)) && rows_ok(k, k_stride, hd, vec) && rows_ok(v, v_stride, hd, vec) &&
        aligned_to(qo, 16) && aligned_to(kc, 16) && aligned_to(vc, 16)) {
        a.gq = cdiv(h, 32 / lph);
        a.gk = cdiv(hkv, 32 / lph);
        const int grid = deal_out(c->sm_count, tokens, a.gq + 2 * a.gk, 3, true, a.deal);
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
