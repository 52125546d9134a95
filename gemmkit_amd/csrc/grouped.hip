// grouped.hip -- bf16 products of ragged groups: the forward product over weights of
// either layout, and the weights' gradient (ragged.h).
#include "ragged.h"

namespace gk {

template <bool BT, EpiKind E>
static hipError_t grouped_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    const int64_t groups = g.G < g.M ? g.G : g.M;
    const int64_t avg = (g.M + groups - 1) / groups;
    if (avg <= 24) return ragged_go<false, false, BT, E, 16, 64, 1, 4, 7>(g, ep, stream);
    if (avg <= 96) return ragged_go<false, false, BT, E, 64, 128, 2, 2, 3>(g, ep, stream);
    return ragged_go<false, false, BT, E, 256, 256, 2, 4, 0>(g, ep, stream);
}

hipError_t launch_grouped_bf16(const RaggedArgs &g, RaggedB bl, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16)
        return bl == RaggedB::Cols ? grouped_go<true, EpiKind::BF16>(g, ep, stream)
                                   : grouped_go<false, EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32)
        return bl == RaggedB::Cols ? grouped_go<true, EpiKind::F32>(g, ep, stream)
                                   : grouped_go<false, EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

template <EpiKind E>
static hipError_t wgrad_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    const int64_t tiles = (int64_t)g.G * ((g.K + 255) / 256) * ((g.N + 255) / 256);
    if (tiles >= g.cus) return ragged_go<false, true, true, E, 256, 256, 2, 4, 0>(g, ep, stream);
    return ragged_go<false, true, true, E, 128, 128, 2, 2, 3>(g, ep, stream);
}

hipError_t launch_grouped_wgrad(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16) return wgrad_go<EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32) return wgrad_go<EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

}  // namespace gk
