// linear.hip -- forward products of linear layers (linear.h).
#include "linear.h"

namespace gk {

hipError_t launch_linear(const RaggedArgs &g, RaggedB bl, EpiKind kind, const LinearParams &p,
                         hipStream_t stream) {
    return linear_launch<false>(g, bl, kind, p, stream);
}

}  // namespace gk
