// grouped.hip -- bf16 products of ragged groups: the forward product over weights of
// either layout, and the weights' gradient (ragged.h).
#include <algorithm>

#include "ragged.h"

namespace gk {

static int64_t avg_rows(const RaggedArgs &g) {
    const int64_t groups = std::min(g.G, g.M);
    return (g.M + groups - 1) / groups;
}

// Products of rows that lack the alignment, in us as rows x groups x k x n with
// k-contiguous / n-contiguous weights, against aligned copies of every group's weights.
bool grouped_takes_any_align(const RaggedArgs &g, RaggedB bl) {
    const int64_t avg = avg_rows(g);
    const double flops = 2.0 * g.M * g.N * g.K;
    // The weights are read once or nearly, those of empty groups not at all: 7x40x2233x5347
    // 24 / 30 against 392 / 481, 1936x56x1285x469 29 / 34 against 47 / 44.
    if (avg <= 64) return true;
    // 13236x82x217x2215 71 / 71 against 91 / 102, 4096x8x1025x1027 30 / 32 against 36 / 34;
    // 16384x8x2049x2047 246 / 246 against 230 / 206
    if (even_tiles(g, avg, 128, 128) >= g.cus) return flops < 6e10;
    // 1001x5x1501x777 18 / 23 against 22 / 22, 5322x16x3633x153 34 / 49 against 57 / 52
    return bl == RaggedB::Rows && flops < 1e10;
}

template <bool BT, EpiKind E>
static hipError_t any_align_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    const int64_t avg = avg_rows(g), stages = ((int64_t)g.K * 2 + 127) / 128;
    const bool few = even_tiles(g, avg, 64, 64) <= g.cus / 2;
    // 4x24x4647x2741 20 / 39 against 42 / 79 with 16 x 64 tiles, 17x55x193x6961 14 / 14
    // against 12 / 12
    if (avg <= 16 && stages < 8 && !few)
        return ragged_go<false, false, BT, E, RegTile<16, 64, 1, 4>>(g, ep, stream);
    if (avg <= 16 || (avg <= 64 && few))
        return ragged_go<false, false, BT, E, RegWaveTile<16, 32, 4>>(g, ep, stream);
    if (avg <= 64) return ragged_go<false, false, BT, E, RegTile<64, 64, 2, 2>>(g, ep, stream);
    if (even_tiles(g, avg, 128, 128) >= g.cus)
        return ragged_go<false, false, BT, E, RegTile<128, 128, 2, 4>>(g, ep, stream);
    if constexpr (!BT) return ragged_go<false, false, BT, E, RegWaveTile<64, 32, 4>>(g, ep, stream);
    return hipErrorInvalidValue;
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

static int64_t wgrad_tiles(const RaggedArgs &g, int side) {
    return (int64_t)g.G * ((g.K + side - 1) / side) * ((g.N + side - 1) / side);
}

// Row ranges per group: a long contraction over few tiles is cut until about two 128 x 128
// tiles per CU have work, each range of 512 rows or more on average.
int wgrad_splits(const RaggedArgs &g) {
    const int64_t avg = g.G > 0 ? g.M / g.G : 0, tiles = wgrad_tiles(g, 128);
    if (avg < 2048 || tiles == 0) return 1;
    const int64_t s = std::min<int64_t>(avg / 512, 2 * g.cus / tiles);
    return (int)std::max<int64_t>(1, std::min<int64_t>(s, 64));
}

// (the figures of both sides: wgrad_go; a longer product repays its copies)
bool wgrad_takes_any_align(const RaggedArgs &g) {
    return g.splits == 1 && 2.0 * g.M * g.N * g.K < 2e10;
}

// Times in us as rows x groups x k x n with f32 / bf16 output.
template <EpiKind E>
static hipError_t wgrad_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    const int64_t cus = g.cus, big = wgrad_tiles(g, 256), avg = g.M / g.G;
    // Rows that lack the alignment as they are, against aligned copies of both operands:
    // 375x5x149x320 9.6 / 9.7 against 14.9 / 13.4, 39x56x513x2409 102 / 58 against
    // 118 / 69 (125 / 82 with 64 x 64 tiles: C's rows lack the alignment too, and long pieces
    // cost less), 4000x8x513x1027 29 / 29 against 32 / 32.
    if (g.any_align) return ragged_go<false, true, true, E, RegTile<64, 128, 2, 2>>(g, ep, stream);
    // The 256 x 256 tile wherever half of the CUs get one: 16384x8x4096x4096 509 / 427 against
    // 675 / 551 with 128 x 128 tiles.  Short groups are bound by the stores, which two
    // workgroups on a CU overlap better, up to four rounds: 1003x32x1024x704 25.4 / 18.8 against
    // 21.7 / 15.5, but 1024x128x2048x512 109 / 66 against 117 / 72.
    if (g.splits == 1 && (big >= 4 * cus || (big >= cus / 2 && avg > 48)))
        return ragged_go<false, true, true, E, BigTile>(g, ep, stream);
    if (g.splits > 1 || avg <= 48)
        return ragged_go<false, true, true, E, RingTile<128, 128, 2, 4, 2>>(g, ep, stream);
    // 4096x4x1024x1024 19.6 / 17.5 against 29.4 / 28.0 with 128 x 128 tiles
    return ragged_go<false, true, true, E, RingTile<64, 64, 2, 2, 3>>(g, ep, stream);
}

hipError_t launch_grouped_wgrad(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16) return wgrad_go<EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32) return wgrad_go<EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

}  // namespace gk
