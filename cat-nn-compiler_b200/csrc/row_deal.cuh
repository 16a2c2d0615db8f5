// How the rows of a kernel's tokens are dealt out to the warps of its grid:
// plain arithmetic without any CUDA type, so that a host compiler takes it too
// and its bounds are checked without a GPU.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define DEAL_FN __host__ __device__ __forceinline__
#else
#define DEAL_FN inline
#endif

namespace catnn {
namespace deal {

typedef int64_t i64;

constexpr int WARPS = 8;  // of a CTA

// A token's row groups go to `parts` warps, `per` to each. Such a team takes
// every teams-th token (run = 0: all warps then read along one front, 17.1 us
// where runs took 18.1 for 16384 tokens of 16 + 4 heads of 64), or a run of
// neighbours, where one look-up serves many (the append: 39 against 43 us).
struct Deal {
    int tokens, groups, parts, per, run, teams;
};
// What one warp of the grid has: groups [g0, g1) of tokens t0, t0 + dt, ... below t1.
struct Share {
    int t0, t1, dt, g0, g1;
};
DEAL_FN Share share_of(const Deal& d, int warp) {
    const int team = warp / d.parts, part = warp - team * d.parts;
    Share s;
    s.t0 = s.t1 = 0;
    if (team < d.teams) {
        if (d.run == 0) {
            s.t0 = team;
            s.t1 = d.tokens;
        } else {
            const i64 t0 = (i64)team * d.run, t1 = t0 + d.run;
            s.t0 = t0 < d.tokens ? (int)t0 : d.tokens;
            s.t1 = t1 < d.tokens ? (int)t1 : d.tokens;
        }
    }
    s.dt = d.run == 0 ? d.teams : 1;
    s.g0 = part * d.per;
    s.g1 = s.g0 + d.per < d.groups ? s.g0 + d.per : d.groups;
    return s;
}

// Deals `groups` row groups of each of `tokens` tokens (both at least 1) out
// to at most sms·per_sm CTAs -> their number. A warp takes all groups of its
// tokens (whose sines and places are then found once a token) unless that
// would leave SMs without warps; a token with more groups than the grid has
// warps gives each warp as many as it takes for the grid to hold one team.
inline int deal_out(int sms, i64 tokens, int groups, int per_sm, bool runs, Deal& d) {
    const i64 want = (i64)sms * 16, most = (i64)sms * per_sm;
    const auto least = [](i64 a, i64 b) { return a < b ? a : b; };
    const auto up = [](i64 a, i64 b) { return (a + b - 1) / b; };
    i64 per = least(groups, tokens * groups / want);
    if (per < up(groups, most * WARPS)) per = up(groups, most * WARPS);
    d.tokens = (int)tokens;
    d.groups = groups;
    d.per = (int)per;
    d.parts = (int)up(groups, per);  // at most `most` CTAs' warps, so that there is always a team
    const i64 ctas = least(most, up(tokens * d.parts, WARPS));
    d.teams = (int)least(tokens, ctas * WARPS / d.parts);
    d.run = runs ? (int)up(tokens, d.teams) : 0;
    return (int)up((i64)d.teams * d.parts, WARPS);
}

// CTAs of the adjoint: what the SMs hold at once, each walking many tokens,
// because every CTA leaves a row of each weight sum in the workspace. At most
// this many, whatever the form of the rows.
constexpr int ADJOINT_PER_SM = 2;
inline i64 adjoint_rows(int sms, i64 tokens, i64 heads) {
    const i64 most = (i64)sms * ADJOINT_PER_SM;
    return most < tokens * heads ? most : tokens * heads;
}

}  // namespace deal
}  // namespace catnn
