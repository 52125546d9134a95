// mxfp4.hip -- MXFP4: quantization of float matrices to rows of e2m1 codes with an e8m0
// scale per 32 elements and back, and products of such operands, plain and per ragged
// group (ragged.h).
//
// Quantization of a block with largest magnitude m (the rule of the OCP microscaling
// formats, e2m1's largest exponent being 2):
//   e = max(floor(log2 m) - 2, -127),  scale byte e + 127 = max(exponent field of m - 2, 0)
//   code = the e2m1 value nearest x * 2^-e, ties to even, magnitudes above 6 to 6
// which v_cvt_scalef32_pk_fp4_* computes from x and 2^e for two elements at a time.  A
// block that holds a NaN or an infinity gets the scale byte 255, the format's NaN, and
// zero codes.
// Bound: HBM.  Lanes hold 16 bytes of a row side by side, four (bf16) or eight (f32) of them
// a block; their largest magnitude goes round by lane permutations.  14336 x 4096 f32: quantize
// 64 us (4.2 TB/s), dequantize 47 us (5.7 TB/s); 333 x 1000 bf16 2.5 us each.
#include <algorithm>

#include "ragged.h"

namespace gk {

__device__ __forceinline__ float mx_scale(int byte) {  // 2^(byte - 127)
    return __uint_as_float(byte ? (uint32_t)byte << 23 : 0x00400000u);
}

// How a kernel walks the values.
//   Vec   unit k stride, rows 16-byte aligned: 16-byte accesses
//   Elem  anything, eight consecutive k per lane
//   Rows  a lane per row, 32 k each: unit row stride (the transposed matrix)
enum class MxWalk { Vec, Elem, Rows };

template <InType T>
__device__ __forceinline__ float mx_load(const void *p, int64_t at) {
    return T == InType::BF16 ? bf16_widen(((const uint16_t *)p)[at]) : ((const float *)p)[at];
}

// Eight values' codes, in one word.
__device__ __forceinline__ uint32_t mx_codes8(const float v[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}

// The scale byte of a block whose largest magnitude has the bits `top`.
__device__ __forceinline__ int mx_byte(uint32_t top) {
    const int e = (int)(top >> 23);
    return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// Four (f32) or eight (bf16) consecutive values of a row from column k0 (zeros past its
// end): 16 bytes.
template <InType T, MxWalk W, int N>
__device__ __forceinline__ void mx_read(const MxArgs &g, int64_t row, int64_t k0, float *v) {
    if (W == MxWalk::Vec && k0 + N <= g.K) {
        const v4i w = *(const v4i *)((const uint8_t *)g.x + (row * g.rs + k0) * (16 / N));
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = __uint_as_float(N == 4 ? (uint32_t)w[i % 4]
                                          : (uint32_t)w[i / 2 % 4] << (i % 2 ? 0 : 16) & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = k0 + i < g.K ? mx_load<T>(g.x, row * g.rs + (k0 + i) * g.cs) : 0.0f;
    }
}

// A workgroup's four waves walk 2^wl segments of 16 blocks of each of its rows.
struct MxGrid {
    int64_t row, rows;  // this wave's first row, and how far to the next
    int seg, lane;
    __device__ __forceinline__ MxGrid(int wl) {
        const int wave = threadIdx.x >> 6;
        lane = threadIdx.x & 63;
        row = ((int64_t)blockIdx.x << (2 - wl)) + (wave >> wl);
        rows = (int64_t)gridDim.x << (2 - wl);
        seg = ((int)blockIdx.y << wl) + (wave & ((1 << wl) - 1));
    }
};

template <InType T, MxWalk W>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const MxArgs g, int wl) {
    const int64_t nb = (g.K + kMxBlock - 1) / kMxBlock;
    if constexpr (W == MxWalk::Rows) {
        const int lane = threadIdx.x & 63;
        const int64_t bands = (g.rows + 63) / 64;
        for (int64_t it = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < bands * nb;
             it += (int64_t)gridDim.x * 4) {
            const int64_t row = it % bands * 64 + lane, blk = it / bands;
            if (row >= g.rows) continue;
            float v[kMxBlock];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kMxBlock; ++i) {
                const int64_t k = blk * kMxBlock + i;
                v[i] = k < g.K ? mx_load<T>(g.x, row * g.rs + k * g.cs) : 0.0f;
                const uint32_t m = __float_as_uint(v[i]) & 0x7FFFFFFFu;
                top = m > top ? m : top;
            }
            const int byte = mx_byte(top);
            v4i w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = byte == 255 ? 0 : (int)mx_codes8(v + 8 * i, mx_scale(byte));
            *(v4i *)(g.codes + row * g.ld + blk * 16) = w;
            g.scales[row * g.lds + blk] = (uint8_t)byte;
            if (blk == nb - 1)  // the row's bytes past its blocks
                for (int64_t b = nb; b < (nb + 15) / 16 * 16; ++b) g.scales[row * g.lds + b] = 0;
        }
    } else {
        // A load of a wave is 1 KiB of the row: bf16 a segment's 16 blocks at four lanes each,
        // f32 half of them at eight.
        constexpr int N = T == InType::BF16 ? 8 : 4, LB = 32 / N, U = 8 / N;
        const MxGrid w(wl);
        if ((int64_t)w.seg * 16 >= nb) return;
        for (int64_t row = w.row; row < g.rows; row += w.rows) {
            float v[U][N];
#pragma unroll
            for (int u = 0; u < U; ++u)
                mx_read<T, W, N>(g, row, ((int64_t)w.seg * U + u) * 64 * N + w.lane * N, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t m = __float_as_uint(v[u][i]) & 0x7FFFFFFFu;
                    top = m > top ? m : top;
                }
                uint32_t o = __builtin_amdgcn_mov_dpp(top, 0xB1, 0xF, 0xF, true);  // lane ^ 1
                top = o > top ? o : top;
                o = __builtin_amdgcn_mov_dpp(top, 0x4E, 0xF, 0xF, true);           // lane ^ 2
                top = o > top ? o : top;
                if constexpr (LB == 8) {
                    o = __builtin_amdgcn_mov_dpp(top, 0x141, 0xF, 0xF, true);      // 7 - lane % 8
                    top = o > top ? o : top;
                }
                const int byte = mx_byte(top);
                const float scale = mx_scale(byte);
                const int64_t blk = ((int64_t)w.seg * U + u) * (64 / LB) + w.lane / LB;
                uint32_t c = 0;
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    uint32_t h = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, v[u][i], v[u][i + 1], scale, 0);
                    h = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(h, v[u][i + 2], v[u][i + 3], scale, 1);
                    c |= h << (4 * i);
                }
                if (byte == 255) c = 0;
                uint8_t *const at = g.codes + row * g.ld + blk * 16 + w.lane % LB * (N / 2);
                if (blk < nb) {
                    if constexpr (N == 8) *(uint32_t *)at = c;
                    else *(uint16_t *)at = (uint16_t)c;
                }
                // (past the row's blocks: zeros, up to the row's 16 bytes)
                if (w.lane % LB == 0) g.scales[row * g.lds + blk] = (uint8_t)byte;
            }
        }
    }
}

template <InType T, MxWalk W>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const MxArgs g, int wl) {
    const int64_t nb = (g.K + kMxBlock - 1) / kMxBlock;
    auto decode = [](uint32_t w, int byte, float v[8]) {
        const float s = mx_scale(byte);
        const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
        const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
        const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
        const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
        v[0] = p0[0], v[1] = p0[1], v[2] = p1[0], v[3] = p1[1];
        v[4] = p2[0], v[5] = p2[1], v[6] = p3[0], v[7] = p3[1];
        if (byte == 255)
            for (int i = 0; i < 8; ++i) v[i] = __builtin_nanf("");
    };
    auto store1 = [&](int64_t at, float v) {
        if constexpr (T == InType::BF16) ((uint16_t *)g.x)[at] = bf16_rne(v);
        else ((float *)g.x)[at] = v;
    };
    if constexpr (W == MxWalk::Rows) {
        const int lane = threadIdx.x & 63;
        const int64_t bands = (g.rows + 63) / 64;
        for (int64_t it = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < bands * nb;
             it += (int64_t)gridDim.x * 4) {
            const int64_t row = it % bands * 64 + lane, blk = it / bands;
            if (row >= g.rows) continue;
            const v4i w = *(const v4i *)(g.codes + row * g.ld + blk * 16);
            const int byte = g.scales[row * g.lds + blk];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float v[8];
                decode((uint32_t)w[c], byte, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t k = blk * kMxBlock + c * 8 + i;
                    if (k < g.K) store1(row * g.rs + k * g.cs, v[i]);
                }
            }
        }
    } else {
        const MxGrid at(wl);
        const int lane = at.lane;
        const int64_t blk = (int64_t)at.seg * 16 + (lane >> 2), k0 = blk * kMxBlock + (lane & 3) * 8;
        if (k0 >= g.K) return;
        for (int64_t row = at.row; row < g.rows; row += at.rows) {
            const uint32_t w = *(const uint32_t *)(g.codes + row * g.ld + blk * 16 + (lane & 3) * 4);
            float v[8];
            decode(w, g.scales[row * g.lds + blk], v);
            if (W == MxWalk::Vec && k0 + 8 <= g.K) {
                if constexpr (T == InType::BF16) {
                    const v4i o = {(int)bf16x2_rne(v[0], v[1]), (int)bf16x2_rne(v[2], v[3]),
                                   (int)bf16x2_rne(v[4], v[5]), (int)bf16x2_rne(v[6], v[7])};
                    *(v4i *)((uint16_t *)g.x + row * g.rs + k0) = o;
                } else {
                    v4f *p = (v4f *)((float *)g.x + row * g.rs + k0);
                    p[0] = v4f{v[0], v[1], v[2], v[3]};
                    p[1] = v4f{v[4], v[5], v[6], v[7]};
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + i < g.K) store1(row * g.rs + (k0 + i) * g.cs, v[i]);
            }
        }
    }
}

template <InType T, MxWalk W>
static hipError_t mx_go(const MxArgs &g, bool quantize, hipStream_t stream) {
    const int64_t nb = (g.K + kMxBlock - 1) / kMxBlock, segs = (nb + 15) / 16;
    int wl = 0;
    dim3 grid;
    if (W == MxWalk::Rows) {
        grid = dim3((uint32_t)std::min<int64_t>(((g.rows + 63) / 64 * nb + 3) / 4, 1 << 20));
    } else {
        wl = segs >= 4 ? 2 : segs >= 2 ? 1 : 0;
        const int64_t wgs = (g.rows + (4 >> wl) - 1) >> (2 - wl);
        grid = dim3((uint32_t)std::min<int64_t>(wgs, 1 << 20), (uint32_t)((segs + (1 << wl) - 1) >> wl));
    }
    if (quantize)
        hipLaunchKernelGGL((mx_quantize_kernel<T, W>), grid, dim3(256), 0, stream, g, wl);
    else
        hipLaunchKernelGGL((mx_dequantize_kernel<T, W>), grid, dim3(256), 0, stream, g, wl);
    return hipGetLastError();
}

template <InType T>
static hipError_t mx_walk(const MxArgs &g, bool quantize, hipStream_t stream) {
    const int64_t esz = (int64_t)in_size(T);
    if (g.cs == 1 && (uintptr_t)g.x % 16 == 0 && (g.rows == 1 || g.rs * esz % 16 == 0))
        return mx_go<T, MxWalk::Vec>(g, quantize, stream);
    const int64_t rs = g.rs < 0 ? -g.rs : g.rs, cs = g.cs < 0 ? -g.cs : g.cs;
    if (g.rows > 1 && rs < cs) return mx_go<T, MxWalk::Rows>(g, quantize, stream);
    return mx_go<T, MxWalk::Elem>(g, quantize, stream);
}

hipError_t launch_mxfp4_quantize(InType in, const MxArgs &g, hipStream_t stream) {
    return in == InType::BF16 ? mx_walk<InType::BF16>(g, true, stream)
                              : mx_walk<InType::F32>(g, true, stream);
}

hipError_t launch_mxfp4_dequantize(InType out, const MxArgs &g, hipStream_t stream) {
    return out == InType::BF16 ? mx_walk<InType::BF16>(g, false, stream)
                               : mx_walk<InType::F32>(g, false, stream);
}

RaggedPlan mxfp4_plan(const RaggedArgs &g) {
    return forward_tile<true, false>(g, [](auto t) { return plan_of(t); });
}

hipError_t launch_mxfp4(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16) return ragged_forward<true, false, EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32) return ragged_forward<true, false, EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

}  // namespace gk
