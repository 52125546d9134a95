// mxint8.hip -- MXINT8, the 8-bit checkpoints of activations: quantization of float matrices
// to rows of int8 codes with an e8m0 scale per 32 elements, and back, through an activation
// where one is given (linear.h).
//
// Quantization of a block with largest magnitude m: e = max(floor(log2 m), -120), step
// 2^(e - 6), scale byte e + 127, code = the whole number nearest x / step, ties to even, at
// most 127 either way: a value is off by half a step (2^-7 of m's power of two), one that would
// round to 128 by up to a whole one.  A block that holds a NaN or an infinity gets the scale byte
// 255 and zero codes.  Values are exact in bf16 and f32.
#include <algorithm>

#include "linear.h"

namespace gk {

// The matrix as rows of CPR chunks of 16 bytes of x (8 bf16, 4 f32), whole blocks, one after the
// other; a workgroup takes 256*U of them in order.
template <int CH>
struct ChunkAt {
    int64_t row;
    int col;
    __device__ __forceinline__ ChunkAt(int64_t row0, uint32_t c0, uint32_t i, uint32_t cpr) {
        const uint32_t c = c0 + i, r = c / cpr;
        row = row0 + r;
        col = (int)(c - r * cpr) * CH;
    }
};

template <InType T, int U>
__global__ __launch_bounds__(256) void mxint8_quantize_kernel(const MxArgs g, uint32_t cpr) {
    constexpr bool F32 = T == InType::F32;
    constexpr int CH = F32 ? 4 : 8, LB = 32 / CH;
    const int64_t first = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = first / cpr;
    const uint32_t c0 = (uint32_t)(first - row0 * cpr);
    v4u raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const ChunkAt<CH> at(row0, c0, threadIdx.x + u * 256, cpr);
        raw[u] = v4u{};
        if (at.row < g.rows && at.col < g.K)
            raw[u] = read_raw<F32, CH>(g.x, at.row * g.rs + at.col * g.cs, g.cs, (int)g.K - at.col);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const ChunkAt<CH> at(row0, c0, threadIdx.x + u * 256, cpr);
        float f[CH];
        widen<F32, CH>(raw[u], f);
        const int byte = mxint8_byte(block_max<LB>(top_bits(f)));
        if (at.row >= g.rows) continue;
        uint8_t *q = g.codes + at.row * g.ld + at.col;
        if constexpr (CH == 8)
            *(v2u *)q = v2u{mxint8_codes4(f, byte), mxint8_codes4(f + 4, byte)};
        else
            *(uint32_t *)q = mxint8_codes4(f, byte);
        if ((at.col & 31) == 0) {
            uint8_t *const s = g.scales + at.row * g.lds + (at.col >> 5);
            *s = (uint8_t)byte;
            // (zeros up to the row's whole 16 bytes)
            if (at.col + 32 >= g.K)
                for (int b = (at.col >> 5) + 1; b & 15; ++b) s[b - (at.col >> 5)] = 0;
        }
    }
}

template <InType T, int U>
__global__ __launch_bounds__(256) void mxint8_dequantize_kernel(const MxArgs g, uint32_t cpr, int act,
                                                                float slope) {
    constexpr bool F32 = T == InType::F32;
    constexpr int CH = F32 ? 4 : 8;
    const int64_t first = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = first / cpr;
    const uint32_t c0 = (uint32_t)(first - row0 * cpr);
    const bool nt = row_lines(g.x, g.rs * (F32 ? 4 : 2));
    v2u codes[U];
    int byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const ChunkAt<CH> at(row0, c0, threadIdx.x + u * 256, cpr);
        codes[u] = v2u{};
        byte[u] = 0;
        if (at.row < g.rows && at.col < g.K) {
            const uint8_t *q = g.codes + at.row * g.ld + at.col;
            if constexpr (CH == 8) codes[u] = *(const v2u *)q;
            else codes[u][0] = *(const uint32_t *)q;
            byte[u] = g.scales[at.row * g.lds + (at.col >> 5)];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const ChunkAt<CH> at(row0, c0, threadIdx.x + u * 256, cpr);
        if (at.row >= g.rows || at.col >= g.K) continue;
        const float step = mxint8_step(byte[u]);
        float f[CH];
#pragma unroll
        for (int e = 0; e < CH; e += 4) mxint8_values4(codes[u][e / 4], step, f + e);
        act_apply(f, act, slope);
        write_row<F32, CH>(g.x, at.row * g.rs + at.col * g.cs, g.cs, (int)g.K - at.col, nt, f);
    }
}

// Small matrices: a chunk a thread, so that they reach more CUs.
template <InType T, typename F>
static hipError_t mxint8_grid(const MxArgs &g, F f) {
    constexpr int CH = T == InType::F32 ? 4 : 8;
    const int64_t cpr = (g.K + kMxBlock - 1) / kMxBlock * (kMxBlock / CH);
    // (a grid's extent counts threads in 32 bits: up to 2^22 workgroups a launch, in whole rows
    // where there are more)
    const int64_t most = std::max<int64_t>(((int64_t)1024 << 22) / cpr, 1);
    for (int64_t r = 0; r < g.rows; r += most) {
        MxArgs p = g;
        p.rows = std::min(most, g.rows - r);
        p.codes += r * g.ld;
        p.scales += r * g.lds;
        p.x = (uint8_t *)g.x + r * g.rs * (int64_t)in_size(T);
        const int64_t chunks = p.rows * cpr;
        const bool wide = chunks >= (1 << 20);
        const int64_t wgs = (chunks + (wide ? 1023 : 255)) / (wide ? 1024 : 256);
        f(p, dim3((uint32_t)wgs), (uint32_t)cpr, wide);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <InType T>
static hipError_t quantize_go(const MxArgs &g, hipStream_t stream) {
    return mxint8_grid<T>(g, [&](const MxArgs &p, dim3 grid, uint32_t cpr, bool wide) {
        if (wide)
            hipLaunchKernelGGL((mxint8_quantize_kernel<T, 4>), grid, dim3(256), 0, stream, p, cpr);
        else
            hipLaunchKernelGGL((mxint8_quantize_kernel<T, 1>), grid, dim3(256), 0, stream, p, cpr);
    });
}

template <InType T>
static hipError_t dequantize_go(const MxArgs &g, int32_t act, float slope, hipStream_t stream) {
    return mxint8_grid<T>(g, [&](const MxArgs &p, dim3 grid, uint32_t cpr, bool wide) {
        if (wide)
            hipLaunchKernelGGL((mxint8_dequantize_kernel<T, 4>), grid, dim3(256), 0, stream, p, cpr,
                               act, slope);
        else
            hipLaunchKernelGGL((mxint8_dequantize_kernel<T, 1>), grid, dim3(256), 0, stream, p, cpr,
                               act, slope);
    });
}

hipError_t launch_mxint8_quantize(InType in, const MxArgs &g, hipStream_t stream) {
    return in == InType::BF16 ? quantize_go<InType::BF16>(g, stream)
                              : quantize_go<InType::F32>(g, stream);
}

hipError_t launch_mxint8_dequantize(InType out, const MxArgs &g, int32_t act, float slope,
                                    hipStream_t stream) {
    return out == InType::BF16 ? dequantize_go<InType::BF16>(g, act, slope, stream)
                               : dequantize_go<InType::F32>(g, act, slope, stream);
}

}  // namespace gk
