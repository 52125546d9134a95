// grouped.hip -- bf16 products of ragged groups: the forward product over weights of
// either layout, and the weights' gradient (ragged.h).
#include <algorithm>

#include "ragged.h"

namespace gk {

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Forward products of rows that lack the alignment, k-contiguous and n-contiguous weights.
// The constants are the least-squares fit of log times of 215 products (1..16384 rows, 1..128
// groups, k and n 128..8192, odd ones among them); the tile they pick, or aligned copies where
// those are expected to cost less, took 1.027 times the fastest of 15 tiles and the copies in
// the geometric mean.
constexpr TileTime kAnyTile[2][5] = {
    {{128, 128, 2.36, 0.839, 2.81, 0.722, 5.90, 0.41},
     {128, 64, 1.57, 0.610, 1.20, 0.463, 7.28, 0.38},
     {32, 64, 1.53, 0.489, 0.28, 0.249, 5.62, 0.00},
     {16, 32, 1.70, 0.169, 0.36, 0.107, 6.62, 0.02},
     {16, 32, 2.15, 0.098, 1.79, 0.091, 6.37, 0.32}},
    {{128, 128, 1.67, 1.247, 2.85, 0.634, 7.16, 0.07},
     {128, 64, 1.18, 0.794, 1.64, 0.453, 7.28, 0.16},
     {32, 64, 0.53, 0.850, 0.26, 0.231, 6.29, 0.00},
     {16, 32, 1.32, 0.285, 0.25, 0.149, 5.52, 0.60},
     {16, 32, 1.81, 0.168, 1.10, 0.155, 6.31, 0.58}}};

bool grouped_plan_any(RaggedArgs &g, RaggedB bl, int64_t copies) {
    const int64_t groups = std::min(g.G, g.M), avg = ceil_div(g.M, groups);
    const int64_t kbytes = (int64_t)g.K * 2;
    const double bytes = ((double)groups * g.N + g.M) * (double)kbytes + 2.0 * g.M * g.N;
    double cost = 0;
    for (int i = 0; i < 5; ++i) {
        const TileTime &t = kAnyTile[bl == RaggedB::Cols ? 1 : 0][i];
        const double tm = groups == 1 ? (double)ceil_div(avg, t.bm)
                                      : std::max(1.0, (double)avg / t.bm + 0.5);
        const double c = tile_time(t, groups * tm * (double)ceil_div(g.N, t.bn) / std::max(g.cus, 1),
                                   (double)ceil_div(kbytes, 128), bytes);
        if (i == 0 || c < cost) {
            g.tile = i;
            cost = c;
        }
    }
    if (avg <= 16) return true;  // the weights are read once, those of empty groups not at all
    double aligned = 0;
    ragged_best<false>(g, groups, avg, ceil_div(kbytes, 16) * 16, &aligned);
    return cost < 4.6 + (double)copies / 2.49e6 + aligned;
}

template <bool BT, EpiKind E>
static hipError_t any_align_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    return any_align_tile(
        g, [&](auto t) { return ragged_go<false, false, BT, PlainOut<E>, decltype(t)>(g, ep, stream); });
}

RaggedPlan grouped_plan(const RaggedArgs &g, RaggedB bl) {
    const auto plan = [](auto t) { return plan_of(t); };
    if (g.any_align) return any_align_tile(g, plan);
    return bl == RaggedB::Cols ? forward_tile<false, true>(g, plan)
                               : forward_tile<false, false>(g, plan);
}

hipError_t launch_grouped_bf16(const RaggedArgs &g, RaggedB bl, const EpiParams &ep,
                               hipStream_t stream) {
    const bool cols = bl == RaggedB::Cols;
    if (g.any_align) {
        if (ep.kind == EpiKind::BF16)
            return cols ? any_align_go<true, EpiKind::BF16>(g, ep, stream)
                        : any_align_go<false, EpiKind::BF16>(g, ep, stream);
        if (ep.kind == EpiKind::F32)
            return cols ? any_align_go<true, EpiKind::F32>(g, ep, stream)
                        : any_align_go<false, EpiKind::F32>(g, ep, stream);
        return hipErrorInvalidValue;
    }
    if (ep.kind == EpiKind::BF16)
        return cols ? ragged_forward<false, true, EpiKind::BF16>(g, ep, stream)
                    : ragged_forward<false, false, EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32)
        return cols ? ragged_forward<false, true, EpiKind::F32>(g, ep, stream)
                    : ragged_forward<false, false, EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

// Weight gradients: aligned operands, and rows that lack the alignment.  Fitted as above to
// 310 aligned products (among them 90 of 700 rows a group and more) and 250 others, f32 and
// bf16 output, with groups whole and cut into 2..16 ranges; what they pick took 1.032 and
// 1.028 times the fastest of all tiles, ranges and copies.  (256 x 256's a and 64 x 64's c2
// are above the fit, 8.01 and 0.170: 1.038 with those.)
constexpr TileTime kWgradTile[2][5] = {
    {{256, 256, 10.0, 1.798, 6.14, 1.099, 5.61, 0.83},
     {128, 128, 5.74, 0.899, 1.36, 0.426, 7.02, 0.00},
     {64, 64, 5.22, 0.217, 0.72, 0.190, 7.28, 0.61},
     {64, 128, 5.34, 0.678, 0.86, 0.238, 7.28, 0.00},
     {32, 64, 5.37, 0.135, 2.37, 0.203, 3.58, 0.63}},
    {{64, 64, 4.65, 1.358, 0.50, 0.330, 5.52, 0.00},
     {128, 128, 5.18, 1.940, 1.40, 0.865, 5.72, 0.37}}};

void wgrad_plan(RaggedArgs &g, EpiKind out, bool can_any, int64_t copies) {
    const double elems = (double)g.G * g.K * g.N, read = 2.0 * g.M * ((double)g.K + g.N);
    const int osz = out == EpiKind::F32 ? 4 : 2;
    const int64_t avg = g.G > 0 ? g.M / g.G : 0;
    double best = 0;
    bool first = true;
    for (int any = 0; any <= (can_any ? 1 : 0); ++any)
        for (int i = 0; i < (any ? 2 : 5); ++i)
            // A long contraction over few tiles is cut into ranges of 128 rows or more, up to
            // four tiles per CU: partial sums in f32, then one launch that adds them.
            for (int s = 1; s <= 16; s *= 2) {
                const TileTime &t = kWgradTile[any][i];
                const double tiles = (double)g.G * ceil_div(g.K, t.bm) * ceil_div(g.N, t.bn) * s;
                if (s > 1 && (avg < s * 128 || tiles > 4.0 * g.cus)) break;
                double c = tile_time(t, tiles / std::max(g.cus, 1),
                                     (double)g.M / std::max(g.G, 1) / 64 / s + 0.5,
                                     read + elems * s * (s > 1 ? 4 : osz));
                if (s > 1) c += 4.0 + elems * (4 * s + osz) / 5e6;
                if (!any && copies > 0) c += 6.0 + (double)copies / 1.89e6;
                if (first || c < best) {
                    first = false;
                    best = c;
                    g.tile = i;
                    g.splits = s;
                    g.any_align = any;
                }
            }
}

template <typename F>
static auto wgrad_tile(const RaggedArgs &g, F f) {
    if (g.any_align) {
        if (g.tile == 0) return f(RegTile<64, 64, 2, 2>{});
        return f(RegTile<128, 128, 2, 4>{});
    }
    switch (g.tile) {
    case 0: return f(BigTile{});
    case 1: return f(RingTile<128, 128, 2, 4, 2>{});
    case 2: return f(RingTile<64, 64, 2, 2, 3>{});
    case 3: return f(RingTile<64, 128, 2, 2, 2>{});
    default: return f(WaveTile<32, 64, 4, 2>{});
    }
}

template <EpiKind E>
static hipError_t wgrad_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    return wgrad_tile(
        g, [&](auto t) { return ragged_go<false, true, true, PlainOut<E>, decltype(t)>(g, ep, stream); });
}

RaggedPlan grouped_wgrad_plan(const RaggedArgs &g) {
    return wgrad_tile(g, [](auto t) { return plan_of(t); });
}

hipError_t launch_grouped_wgrad(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16) return wgrad_go<EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32) return wgrad_go<EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

}  // namespace gk
