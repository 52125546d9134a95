// grouped.hip -- bf16 products of ragged groups: the forward product over weights of
// either layout, and the weights' gradient (ragged.h).
#include <algorithm>

#include "ragged.h"

namespace gk {

hipError_t launch_grouped_bf16(const RaggedArgs &g, RaggedB bl, const EpiParams &ep,
                               hipStream_t stream) {
    const bool cols = bl == RaggedB::Cols;
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

// Times in us as rows x groups x k x n with f32 / bf16 output.
template <EpiKind E>
static hipError_t wgrad_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    const int64_t cus = g.cus, big = wgrad_tiles(g, 256), avg = g.M / g.G;
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
