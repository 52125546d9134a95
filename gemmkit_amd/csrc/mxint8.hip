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

// ONCE: x of whole chunks, nontemporally and without a branch around a load (kernels, us, plain loads
// / so: bf16 16384 x 4096 51 / 40.4 (5.1 TB/s), 8192 x 4096 28.7 / 19.6, f32 16384 x 4000 91.7 / 64.6;
// nontemporally 4096 x 4096 loses, 10.8 / 11.9).
template <InType T, int U, bool ONCE>
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
        const bool in = at.row < g.rows && at.col < g.K;
        raw[u] = v4u{};
        if constexpr (ONCE) {
            typedef v4u v4u_any2 __attribute__((aligned(2)));
            const uint8_t *x = (const uint8_t *)g.x + (in ? at.row * g.rs + at.col : 0) * (F32 ? 4 : 2);
            const v4u v = __builtin_nontemporal_load((const v4u_any2 *)x);
            raw[u] = in ? v : v4u{};
        } else if (in) {
            raw[u] = read_raw<F32, CH>(g.x, at.row * g.rs + at.col * g.cs, g.cs, (int)g.K - at.col);
        }
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

// ---------------------------------------------------------------- weight gradient

// A's stages of a weight gradient whose left operand is a checkpoint: loaded as codes, and put in
// the stage as act(values), rounded to bf16: what the bf16 instructions take.  Their rounding, half of 2^-7 of a value's power of two, is
// at most the checkpoint's own, half of 2^-6 of its block's largest: 1003x1024x704 through GELU is
// off by 0.0019 of its norm where f32 activations would leave 0.0017 (bf16 output).  (RegPanel's
// transposed stage; each thread decodes LP chunks of eight values a stage, once for every tile of its
// columns.)
template <int W, int NW>
struct CodePanel {
    static constexpr int BYTES = W * 128, NI = BYTES / 1024, LP = NI / NW;
    static_assert(NI % NW == 0, "every wave has chunks");
    static constexpr int kNone = INT32_MAX;
    static constexpr bool CODES = true;
    using Reg = v4i;  // eight codes, their scale byte
    const uint8_t *codes, *scales;  // of the next stage
    int ld, lds, left, act;
    float slope;
    uint32_t vc[LP], vs[LP];  // this lane's offsets from them
    int pos[LP];              // its rows, kNone: outside the tile
    int wave, lane;

    __device__ __forceinline__ void init(const RaggedArgs &g, const RaggedTile &t, int wave_, int lane_) {
        codes = uniform((const uint8_t *)g.a + t.row0);
        scales = uniform(g.sa + (t.row0 >> 5));
        ld = (int)g.lda;
        lds = (int)g.lsa;
        left = t.k;
        act = g.act;
        slope = g.slope;
        wave = wave_;
        lane = lane_;
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            const int at = (wave * LP + i) * 64 + lane, row = at / (W / 8), slot = at % (W / 8);
            const int c = ((((slot >> 1) ^ tr_unit<W>(row)) << 1) | (slot & 1)) * 8;  // column
            vc[i] = (uint32_t)(row * ld + c);
            vs[i] = (uint32_t)(row * lds + (c >> 5));
            pos[i] = c < t.rows ? row : kNone;
        }
    }
    __device__ __forceinline__ void load(Reg (&r)[LP]) const {
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            v4i v = {};
            if (pos[i] < left) {
                const v2i w = *(const v2i *)(codes + vc[i]);
                v = v4i{w[0], w[1], scales[vs[i]], 0};
            }
            r[i] = v;
        }
    }
    __device__ __forceinline__ void skip(int stages) {
        codes += (int64_t)stages * 64 * ld;
        scales += (int64_t)stages * 64 * lds;
        left -= stages * 64;
    }
    __device__ __forceinline__ void store(const Reg (&r)[LP], uint8_t *dst) const {
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            const float step = mxint8_step(r[i][2]);
            float f[8];
            mxint8_values4((uint32_t)r[i][0], step, f);
            mxint8_values4((uint32_t)r[i][1], step, f + 4);
            act_apply(f, act, slope);
            const v4i v = {(int)bf16x2_rne(f[0], f[1]), (int)bf16x2_rne(f[2], f[3]),
                           (int)bf16x2_rne(f[4], f[5]), (int)bf16x2_rne(f[6], f[7])};
            *(v4i *)(dst + (wave * LP + i) * 1024 + lane * 16) = v;
        }
    }
};

template <EpiKind E>
static hipError_t wgrad8_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    constexpr int BM = 64, BN = 64;
    const int64_t per = (int64_t)((g.K + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    // (32-bit offsets inside a stage of 64 rows)
    if (per > INT32_MAX / 16 || 64 * std::max(std::max(g.lda, g.lsa), g.ldb) > (int64_t)kMaxRecords)
        return hipErrorInvalidValue;
    hipLaunchKernelGGL((ragged_reg_kernel<true, true, PlainOut<E>, BM, BN, 2, 2, CodePanel<BM, 4>>),
                       ragged_grid((int64_t)wgrad_share((int)per) * 8), dim3(256), 0, stream, g, ep);
    return hipGetLastError();
}

// Few rows and tiles.  Traced kernels / calls one after the other, us, decoded in the tiles against
// decoded first (two launches and a workspace): 64x1024x704 5.3 / 8.8 against 6.5 / 14.8, 256x1024x704
// 7.3 / 8.7 against 7.2 / 14.8, 512x1024x704 10.2 / 9.4 against 8.3 / 14.8; through GELU 64 rows 6.6 / 8.8
// against 6.8 / 14.8, 128 rows 8.0 / 8.8 against 6.9 / 14.8, 256 rows 10.7 / 9.8 against 7.5 / 14.9 (each
// tile of a column computes it again).  The bounds lie where a device that other work keeps busy, to
// which the kernels' times count, loses no more than 1 us; one that waits for the host gains 6.
bool wgrad8_direct(const RaggedArgs &g) {
    const int64_t tiles = (int64_t)((g.K + 63) / 64) * ((g.N + 63) / 64);
    const bool smooth = g.act != kActNone && g.act != kActRelu && g.act != kActLeakyRelu;
    return g.M <= (smooth ? 128 : 256) && tiles <= 2 * (int64_t)g.cus;
}

hipError_t launch_wgrad8(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    if (ep.kind == EpiKind::BF16) return wgrad8_go<EpiKind::BF16>(g, ep, stream);
    if (ep.kind == EpiKind::F32) return wgrad8_go<EpiKind::F32>(g, ep, stream);
    return hipErrorInvalidValue;
}

// ---------------------------------------------------------------- launch

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
    const bool once = g.rows * g.K * (int64_t)in_size(T) >= kOnceBytes && g.cs == 1 &&
                      g.K % (T == InType::F32 ? 4 : 8) == 0;
    return mxint8_grid<T>(g, [&](const MxArgs &p, dim3 grid, uint32_t cpr, bool wide) {
        if (wide && once)
            hipLaunchKernelGGL((mxint8_quantize_kernel<T, 4, true>), grid, dim3(256), 0, stream, p, cpr);
        else if (wide)
            hipLaunchKernelGGL((mxint8_quantize_kernel<T, 4, false>), grid, dim3(256), 0, stream, p, cpr);
        else
            hipLaunchKernelGGL((mxint8_quantize_kernel<T, 1, false>), grid, dim3(256), 0, stream, p, cpr);
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
