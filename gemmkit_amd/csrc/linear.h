#pragma once
// linear.h -- what a linear layer's products do on their way out of the accumulators:
// bias, activation, residual and the pre-activation kept for the backward pass; or, in the
// backward pass, the activation's derivative and the bias gradient.
//
// Activations and derivatives, with P(z) the normal distribution and p(z) its density:
//   gelu       z P(z)                 P + z p
//   gelu_tanh  z s, s = sigmoid(2u)   s + z s (1 - s) 2u',  u = c (z + 0.044715 z^3), c^2 = 2/pi
//   silu       z s, s = sigmoid(z)    s + z s (1 - s)
// GELU is max(z, 0) - a P(-a) with a = |z|, and P(-a) = exp(-a^2/2) t r(t), t = 1 / (1 + 0.3 a), with
// the polynomial r of degree 7 whose largest error relative to P is least on [0, 13.5], where f32 ends
// (a linear program over 600 points: 1.3e-7): the tail keeps its own leading bits, and GELU its sign.
// (A polynomial times the exponential, without the reciprocal, is off by 3e-7 of 1, wrong in sign
// beyond -5, and saves 1%: 8192 x 4096 x 8192 with GELU 430 us against 434, its gradient 444 against 451.)
#include "ragged.h"

namespace gk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluC2 = 1.5957691216057308f;  // 2 sqrt(2/pi)
constexpr float kGeluCubic = 0.044715f;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// P(-a) - SLOPE a p(a) (SLOPE 0 or 1) for a = |z|, at most 13.5 (beyond it the exponential is 0).
template <int SLOPE>
__device__ __forceinline__ float normal_tail(float z, float a) {
    constexpr float kDensity = 0.3989422804f;  // 1 / sqrt(2 pi)
    const float e = fast_exp2(z * z * (-0.5f * kLog2e));
    const float t = fast_rcp(__builtin_fmaf(a, 0.3f, 1.0f));
    float q = 3.593174368e-02f;
    q = __builtin_fmaf(q, t, -1.582760066e-01f);
    q = __builtin_fmaf(q, t, 2.082066089e-01f);
    q = __builtin_fmaf(q, t, -5.539386347e-02f);
    q = __builtin_fmaf(q, t, 1.294692159e-01f);
    q = __builtin_fmaf(q, t, 9.963748604e-02f);
    q = __builtin_fmaf(q, t, 1.207983643e-01f);
    q = __builtin_fmaf(q, t, 1.196263954e-01f);
    q *= t;
    if (SLOPE) q = __builtin_fmaf(a, -kDensity, q);
    return q * e;
}
__device__ __forceinline__ float normal_clamp(float z) {
    return __builtin_fminf(__builtin_fabsf(z), 13.5f);
}

__device__ __forceinline__ float sigmoid(float z) {
    return fast_rcp(1.0f + fast_exp2(-kLog2e * z));
}
__device__ __forceinline__ float gelu_inner(float z) {
    return z * __builtin_fmaf(kGeluC2 * kGeluCubic, z * z, kGeluC2);
}

// f = act(f).  NaN stays NaN, through ReLU and LeakyReLU too (unlike fused_apply's): a checkpoint's
// mark of an overflow is to be seen behind them.  Their -0 gives 0.
template <int N>
__device__ __forceinline__ void act_apply(float (&f)[N], int act, float slope) {
    if (act == kActGelu) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float a = normal_clamp(f[e]);
            f[e] = __builtin_fmaf(-a, normal_tail<0>(f[e], a), __builtin_fmaxf(f[e], 0.0f));
        }
    } else if (act == kActGeluTanh) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= sigmoid(gelu_inner(f[e]));
    } else if (act == kActSilu) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= sigmoid(f[e]);
    } else if (act != kActNone) {
        const float s = act == kActRelu ? 0.0f : slope;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float hi = f[e] <= 0.0f ? 0.0f : f[e], lo = f[e] < 0.0f ? f[e] : 0.0f;
            f[e] = act == kActRelu ? hi : __builtin_fmaf(s, lo, hi);
        }
    }
}

// f *= act'(z); at 0 ReLU's derivative is 0 and LeakyReLU's the slope, at a NaN every one is NaN.
template <int N>
__device__ __forceinline__ void act_scale(float (&f)[N], const float (&z)[N], int act, float slope) {
    if (act == kActGelu) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float w = normal_tail<1>(z[e], normal_clamp(z[e]));
            f[e] *= z[e] > 0.0f ? 1.0f - w : w;
        }
    } else if (act == kActGeluTanh) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            // (s (1 - s) from exp(-|2u|): as 1 - s it would lose what z and u' multiply)
            const float u = gelu_inner(z[e]), t = fast_exp2(-kLog2e * __builtin_fabsf(u));
            const float r = fast_rcp(1.0f + t), q = t * r;
            // (beyond 16 q is 0, and the square would overflow far out)
            const float b = __builtin_amdgcn_fmed3f(z[e], -16.0f, 16.0f);
            const float du = __builtin_fmaf(3.0f * kGeluC2 * kGeluCubic, b * b, kGeluC2);
            f[e] *= __builtin_fmaf(q * r, b * du, u > 0.0f ? r : q);
        }
    } else if (act == kActSilu) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            // (beyond 128 s is 1 or 0: an infinity would make NaN of the limits)
            const float s = sigmoid(z[e]), b = __builtin_amdgcn_fmed3f(z[e], -128.0f, 128.0f);
            f[e] *= s * __builtin_fmaf(b, 1.0f - s, 1.0f);
        }
    } else if (act != kActNone) {
        const float s = act == kActRelu ? 0.0f : slope;
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= z[e] > 0.0f ? 1.0f : z[e] <= 0.0f ? s : z[e];
    }
}

// ---------------------------------------------------------------- MXINT8

// The scale byte of a block whose largest magnitude has the bits `top`.
__device__ __forceinline__ int mxint8_byte(uint32_t top) {
    const int e = (int)(top >> 23);
    return e > kMxint8Min ? e : kMxint8Min;
}
// Four values as codes: nearest whole multiple of the step, ties to even, at most 127.  A
// value times 1/step is below 2^7, and 1.5 * 2^23 added to it leaves the whole number, rounded, in
// the low bits.
__device__ __forceinline__ uint32_t mxint8_codes4(const float *v, int byte) {
    constexpr int kOne = 0x4B400000;  // 1.5 * 2^23
    const float inv = __uint_as_float((uint32_t)(260 - byte) << 23);
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = (int)__float_as_uint(__builtin_fmaf(v[i], inv, 12582912.0f));
        c[i] = c[i] < kOne - 127 ? kOne - 127 : c[i];
        c[i] = c[i] > kOne + 127 ? kOne + 127 : c[i];
    }
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)c[1], (uint32_t)c[0], 0x0C0C0400);
    const uint32_t hi = __builtin_amdgcn_perm((uint32_t)c[3], (uint32_t)c[2], 0x04000C0C);
    return byte == 255 ? 0 : lo | hi;
}
// The bits of the largest magnitude of N values; a NaN's where one is a NaN.
template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&v)[N]) {
    float m = __builtin_fabsf(v[0]);
#pragma unroll
    for (int e = 1; e < N; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[e]));
    return __float_as_uint(m) & 0x7FFFFFFFu;
}
__device__ __forceinline__ float mxint8_step(int byte) {
    return byte == 255 ? __builtin_nanf("") : __builtin_ldexpf(1.0f, byte - 133);
}
__device__ __forceinline__ void mxint8_values4(uint32_t w, float step, float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)((int32_t)(w << (24 - 8 * i)) >> 24) * step;
}
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }
// The largest of `top` over the LB lanes (4 or 8) of a block.
template <int LB>
__device__ __forceinline__ uint32_t block_max(uint32_t top) {
    top = max_bits(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
    top = max_bits(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
    if constexpr (LB == 8)
        top = max_bits(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x141, 0xF, 0xF, true));  // 7 - lane % 8
    return top;
}

// ---------------------------------------------------------------- output

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// CH consecutive bf16 or f32 values of a row at p (element stride cs; cols of them, at least one,
// exist), as they lie in memory.  (Alone they are loaded without branches, values past the last
// one from there: behind branches each load would wait for the one before it.)
template <bool F32, int CH>
__device__ __forceinline__ v4u read_raw(const void *p, int64_t at, int64_t cs, int cols) {
    v4u w = {};
    if constexpr (F32) {
        static_assert(CH == 4, "16 bytes");
        typedef v4u v4u_any4 __attribute__((aligned(4)));
        const uint32_t *q = (const uint32_t *)p + at;
        if (cs == 1 && cols >= CH) return *(const v4u_any4 *)q;
        uint32_t v[CH];
#pragma unroll
        for (int e = 0; e < CH; ++e) v[e] = q[(e < cols ? e : cols - 1) * cs];
#pragma unroll
        for (int e = 0; e < CH; ++e) w[e] = e < cols ? v[e] : 0;
    } else {
        const uint16_t *q = (const uint16_t *)p + at;
        if (cs == 1 && cols >= CH) {
            if constexpr (CH == 8) {
                typedef v4u v4u_any2 __attribute__((aligned(2)));
                return *(const v4u_any2 *)q;
            } else {
                const v2u_any2 h = *(const v2u_any2 *)q;
                w[0] = h[0];
                w[1] = h[1];
                return w;
            }
        }
        uint16_t v[CH];
#pragma unroll
        for (int e = 0; e < CH; ++e) v[e] = q[(e < cols ? e : cols - 1) * cs];
#pragma unroll
        for (int e = 0; e < CH; ++e) w[e / 2] |= e < cols ? (uint32_t)v[e] << (16 * (e % 2)) : 0;
    }
    return w;
}

template <bool F32, int CH>
__device__ __forceinline__ void widen(const v4u &w, float (&f)[CH]) {
#pragma unroll
    for (int e = 0; e < CH; ++e)
        f[e] = __uint_as_float(F32 ? w[e % 4] : e % 2 ? w[e / 2 % 4] & 0xFFFF0000u : w[e / 2 % 4] << 16);
}

// CH values of a row, rounded once; NT: whole lines, stored nontemporally.
template <bool F32, int CH>
__device__ __forceinline__ void write_row(void *p, int64_t at, int64_t cs, int cols, bool nt,
                                          const float (&f)[CH]) {
    v4u w = {};
    if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < CH; ++e) w[e] = __float_as_uint(f[e]);
    } else {
#pragma unroll
        for (int e = 0; e < CH / 2; ++e) w[e] = bf16x2_rne(f[2 * e], f[2 * e + 1]);
    }
    if (cs == 1 && cols >= CH) {
        typedef v4u v4u_any2 __attribute__((aligned(2)));
        if constexpr (CH * (F32 ? 4 : 2) == 16) {
            v4u_any2 *q = (v4u_any2 *)((uint8_t *)p + at * (F32 ? 4 : 2));
            if (nt) __builtin_nontemporal_store(w, q);
            else *q = w;
        } else {
            *(v2u_any2 *)((uint16_t *)p + at) = v2u_any2{w[0], w[1]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < CH; ++e)
        if (e < cols) {
            if constexpr (F32) ((uint32_t *)p)[at + e * cs] = w[e];
            else ((uint16_t *)p)[at + e * cs] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
        }
}

__device__ __forceinline__ bool row_lines(const void *p, int64_t row_bytes) {
    return (((uint64_t)p | (uint64_t)row_bytes) & 127) == 0;
}

// Rows of a tile as a buffer: accesses past its rows or columns read zeros and write nothing.
struct Rows {
    __amdgpu_buffer_rsrc_t r;
    uint32_t at, step;  // this lane's offset in the next pass, and from pass to pass
    // base: the tile's first element; width: bytes of the tile's columns; in, col: the lane's
    // column in bytes if it is one of them
    __device__ __forceinline__ Rows(const void *base, int64_t ld, int rows, int width, int row,
                                    int col, bool in, int rpp) {
        const uint8_t *const b = uniform((const uint8_t *)base);
        const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)ld);
        r = __builtin_amdgcn_make_buffer_rsrc(
            (void *)b, (short)0, (int)__builtin_amdgcn_readfirstlane((rows - 1) * l + width),
            kRsrcWord3);
        at = in ? row * l + col : kOutOfRange;
        step = rpp * l;
    }
    // A chunk of CH elements of SZ bytes, of which cols are in the matrix: one by one, zeros for
    // the others.
    template <int CH, int SZ>
    __device__ __forceinline__ void load(uint32_t (&v)[CH], int cols) {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            const uint32_t o = e < cols ? at + e * SZ : kOutOfRange;
            if constexpr (SZ == 4) v[e] = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0);
            else v[e] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0);
        }
        at += step;
    }
    // PART: some chunks of the wave are not whole.
    template <int CH, int SZ, bool PART>
    __device__ __forceinline__ void store(const v4u &w, int cols, bool nt) {
        const uint32_t o = PART && cols < CH ? kOutOfRange : at;
        if constexpr (CH * SZ == 16) {
            if (nt) __builtin_amdgcn_raw_buffer_store_b128(w, r, o, 0, 2);
            else __builtin_amdgcn_raw_buffer_store_b128(w, r, o, 0, 0);
        } else {
            __builtin_amdgcn_raw_buffer_store_b64(v2u{w[0], w[1]}, r, o, 0, 0);
        }
        if constexpr (PART) {
#pragma unroll
            for (int e = 0; e < CH - 1; ++e) {
                const uint32_t p = cols < CH && e < cols ? at + e * SZ : kOutOfRange;
                if constexpr (SZ == 4) __builtin_amdgcn_raw_buffer_store_b32(w[e % 4], r, p, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(w[e / 2] >> (16 * (e % 2))), r, p, 0, 0);
            }
        }
        at += step;
    }
};

// Elements loaded one by one, as they lie in memory.
template <int CH, int SZ>
__device__ __forceinline__ v4u packed(const uint32_t (&v)[CH]) {
    v4u w = {};
#pragma unroll
    for (int e = 0; e < CH; ++e) {
        if constexpr (SZ == 4) w[e % 4] = v[e];
        else w[e / 2] |= v[e] << (16 * (e % 2));
    }
    return w;
}

// Matrices read once from this size on, a quarter of the Infinity Cache, are read nontemporally by the
// kernels that do nothing else; smaller ones may lie in the caches, and lose.
constexpr int64_t kOnceBytes = (int64_t)64 << 20;

// Rows of a product for which sums holds one row: a tile's, or (256 x 256) half a tile's,
// since the last round's tiles may go out as halves.
constexpr int sum_unit(int bm) { return bm == 256 ? 128 : bm; }

// Bands whose inputs are in flight while one is worked on (LinearOut::chunked): 8192 x 4096 x 8192's
// input gradient through a checkpoint 440 us with two, 444 with one; four spill.
constexpr int kAhead = 2;

template <EpiKind E, bool GRAD>
struct LinearOut {
    using Params = LinearParams;
    static constexpr bool F32 = E == EpiKind::F32;
    static constexpr int CH = chunk_of(E);
    static constexpr int LB = 32 / CH;  // lanes of a checkpoint's block

    // What a chunk reads: the residual, or the pre-activations (v) with their scale.
    struct In {
        v4u v;
        int byte;
    };
    __device__ __forceinline__ static In load(const Params &p, int row, int col, int N, bool live) {
        In in = {};
        if (!live || col >= N) return in;
        if constexpr (!GRAD) {
            if (p.res)
                in.v = read_raw<F32, CH>(p.res, row * p.rsr + col * p.csr, p.csr, N - col);
        } else if (p.codes) {
            // (a begun block's codes are all there)
            const uint8_t *q = p.codes + row * p.ld + col;
            if constexpr (CH == 8) {
                const v2u w = *(const v2u *)q;
                in.v[0] = w[0];
                in.v[1] = w[1];
            } else {
                in.v[0] = *(const uint32_t *)q;
            }
            in.byte = p.scales[row * p.lds + (col >> 5)];
        } else if (p.z) {
            in.v = read_raw<false, CH>(p.z, row * p.rsz + col * p.csz, p.csz, N - col);
        }
        return in;
    }
    struct Flags {
        bool nt_c, nt_z;
        __device__ __forceinline__ explicit Flags(const Params &p) {
            nt_c = row_lines(p.c, p.rsc * (F32 ? 4 : 2));
            nt_z = row_lines(p.z, p.rsz * 2);
        }
    };
    __device__ __forceinline__ static void bias_of(const Params &p, int col, int N, float (&b)[CH]) {
#pragma unroll
        for (int e = 0; e < CH; ++e) b[e] = 0.0f;
        if (GRAD || !p.bias) return;
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (col + e < N)
                b[e] = p.bias_f32 ? ((const float *)p.bias)[col + e]
                                  : bf16_widen(((const uint16_t *)p.bias)[col + e]);
    }
    // f: sums of products in; the gradient before rounding out.
    __device__ __forceinline__ static void grad_map(const Params &p, float alpha, int kind,
                                                    const In &in, float (&f)[CH]) {
#pragma unroll
        for (int e = 0; e < CH; ++e) f[e] *= alpha;
        if (kind == 0) return;
        float z[CH];
        if (kind == 2) {
            const float step = mxint8_step(in.byte);
#pragma unroll
            for (int e = 0; e < CH; e += 4) mxint8_values4(in.v[e / 4], step, z + e);
        } else {
            widen<false, CH>(in.v, z);
        }
        act_scale(f, z, p.act, p.slope);
    }
    // f: pre-activations in, the output before rounding out.
    __device__ __forceinline__ static void act_map(const Params &p, bool res, const In &in,
                                                   float (&f)[CH]) {
        act_apply(f, p.act, p.slope);
        if (res) {
            float r[CH];
            widen<F32, CH>(in.v, r);
#pragma unroll
            for (int e = 0; e < CH; ++e) f[e] += r[e];
        }
    }
    // The chunk's codes (in w) and its block's scale byte; every lane of the block comes along.
    // (Columns past the matrix are 0, or not finite in a row whose other columns are not either.)
    __device__ __forceinline__ static int quantize(const float (&f)[CH], v2u &w) {
        const int byte = mxint8_byte(block_max<LB>(top_bits(f)));
        w[0] = mxint8_codes4(f, byte);
        w[1] = CH == 8 ? mxint8_codes4(f + CH - 4, byte) : 0;
        return byte;
    }
    // The whole way of a chunk, whatever the views' strides and however few of its columns there
    // are.
    __device__ __forceinline__ static void store(const Params &p, const Flags &fl, int row, int col,
                                                 int N, const float (&bias)[CH], const In &in,
                                                 float (&f)[CH]) {
        const int cols = N - col;  // (0 or less: outside the matrix)
        if constexpr (GRAD) {
            grad_map(p, p.alpha, p.codes ? 2 : p.z ? 1 : 0, in, f);
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) f[e] = __builtin_fmaf(p.alpha, f[e], bias[e]);
            if (p.codes) {
                v2u w;
                const int byte = quantize(f, w);
                if ((col >> 5) < (N + 31) >> 5) {
                    uint8_t *q = p.codes + row * p.ld + col;
                    if constexpr (CH == 8) *(v2u *)q = w;
                    else *(uint32_t *)q = w[0];
                    if ((col & 31) == 0) p.scales[row * p.lds + (col >> 5)] = (uint8_t)byte;
                }
            } else if (p.z && cols > 0) {
                write_row<false, CH>(p.z, row * p.rsz + col * p.csz, p.csz, cols, fl.nt_z, f);
            }
            act_map(p, p.res != nullptr, in, f);
        }
        if (cols > 0) write_row<F32, CH>(p.c, row * p.rsc + col * p.csc, p.csc, cols, fl.nt_c, f);
    }

    // Column sums of a tile from the first row of its unit on.
    template <int BM>
    __device__ __forceinline__ static void put_sum(const Params &p, const RaggedTile &t, int N,
                                                   int c, float s) {
        constexpr int UNIT = sum_unit(BM);
        if (t.n0 + c >= N) return;
        float *q = p.sums + (int64_t)(t.row0 / UNIT) * N + t.n0 + c;
        q[0] = s;
        if (UNIT < BM && t.rows > UNIT) q[N] = 0.0f;
    }

    // What a tile reads beside its products, the chunks of each thread of a tile that goes out by
    // slabs() and of each lane of one that goes out by bands, in registers before the
    // products are done where they are few.
    template <int BM, int BN, int THREADS>
    struct EarlySlab {
        static constexpr int CPR = BN / CH, CHUNKS = BM * CPR, U = (CHUNKS + THREADS - 1) / THREADS;
        In in[U];
        float bias[U][CH];
        __device__ __forceinline__ void load(const Params &p, const RaggedTile &t, int N, int, int) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = threadIdx.x + u * THREADS, row = c / CPR, col = t.n0 + c % CPR * CH;
                const bool live = c < CHUNKS && row < t.rows;
                in[u] = LinearOut::load(p, t.row0 + row, col, N, live);
                bias_of(p, live ? col : N, N, bias[u]);
            }
        }
    };
    template <int BM, int BN, int WM, int WN>
    struct EarlyBands {
        static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, CPR = WTN / CH;
        static constexpr int RPP = 64 / CPR, P = 16 / RPP;
        static constexpr bool ALL = TM * P <= 4;
        In in[ALL ? TM * P : 1];
        float bias[ALL ? CH : 1];
        __device__ __forceinline__ void load(const Params &p, const RaggedTile &t, int N, int wave,
                                             int lane) {
            if constexpr (ALL) {
                const int col = t.n0 + wave % WN * WTN + lane % CPR * CH;
#pragma unroll
                for (int i = 0; i < TM * P; ++i) {
                    const int row = wave / WN * WTM + i * RPP + lane / CPR;
                    in[i] = LinearOut::load(p, t.row0 + row, col, N, row < t.rows);
                }
                bias_of(p, col, N, bias);
            }
        }
    };
    template <int BM, int BN, int WM, int WN>
    using EarlyTile = std::conditional_t<(BN / WN < 32), EarlySlab<BM, BN, WM * WN * 64>,
                                         EarlyBands<BM, BN, WM, WN>>;
    template <int BM, int BN, int KS>
    using EarlyWaves = EarlySlab<BM, BN, KS * 64>;

    // Tiles that lie in LDS whole, SLABS partial sums of each element one after the other, of
    // which every thread takes chunks.
    template <int BM, int BN, int THREADS, int SLABS>
    __device__ __forceinline__ static void slabs(const Params &p, const RaggedTile &t, int N,
                                                 float *sums,
                                                 const EarlySlab<BM, BN, THREADS> &early) {
        constexpr int LD = BN + 4, CPR = BN / CH, CHUNKS = BM * CPR;
        constexpr int U = EarlySlab<BM, BN, THREADS>::U;
        static_assert(CHUNKS % 64 == 0 && BN % 32 == 0, "whole waves, whole blocks");
        const Flags fl(p);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = threadIdx.x + u * THREADS, row = c / CPR, at = c % CPR * CH;
            if (c >= CHUNKS || row >= t.rows) continue;
            float f[CH];
#pragma unroll
            for (int i = 0; i < CH; i += 4) {
                v4f v = {};
#pragma unroll
                for (int w = 0; w < SLABS; ++w) v += *(const v4f *)(sums + (w * BM + row) * LD + at + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[i + e] = v[e];
            }
            store(p, fl, t.row0 + row, t.n0 + at, N, early.bias[u], early.in[u], f);
            if (GRAD && p.sums) {
#pragma unroll
                for (int i = 0; i < CH; i += 4)
                    *(v4f *)(sums + row * LD + at + i) = v4f{f[i], f[i + 1], f[i + 2], f[i + 3]};
            }
        }
        if (GRAD && p.sums) {
            __syncthreads();
            for (int c = threadIdx.x; c < BN; c += THREADS) {
                float s = 0.0f;
                for (int r = 0; r < t.rows; ++r) s += sums[r * LD + c];
                put_sum<BM>(p, t, N, c, s);
            }
        }
    }

    template <int BM, int BN, int KS, int SMEM, int TM, int TN>
    __device__ __forceinline__ static void waves(const Params &p, const RaggedTile &t, int N,
                                                 const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                                 int lane, const EarlyWaves<BM, BN, KS> &early) {
        constexpr int LD = BN + 4;
        static_assert(KS * BM * LD * 4 <= SMEM, "LDS");
        float *const sums = (float *)smem;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                *(v4f *)(sums + (wave * BM + i * 16 + (lane & 15)) * LD + j * 16 + 4 * (lane >> 4)) =
                    acc[i][j];
        slabs<BM, BN, KS * 64, KS>(p, t, N, sums, early);
    }

    template <int BM, int BN, int WM, int WN, int SMEM, int TM, int TN>
    __device__ __forceinline__ static void tile(const Params &p, const RaggedTile &t, int N,
                                                const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                                int lane, const EarlyTile<BM, BN, WM, WN> &early) {
        constexpr int WTM = BM / WM, WTN = BN / WN;
        const int wm = wave / WN, wn = wave % WN, l16 = lane & 15, lq = lane >> 4;
        if constexpr (WTN < 32) {
            // A wave's columns are no whole block of a checkpoint: the tile goes through LDS
            // whole.
            constexpr int LD = BN + 4;
            static_assert(BM * LD * 4 <= SMEM, "LDS");
            float *const sums = (float *)smem;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    *(v4f *)(sums + (wm * WTM + i * 16 + l16) * LD + wn * WTN + j * 16 + 4 * lq) =
                        acc[i][j];
            slabs<BM, BN, WM * WN * 64, 1>(p, t, N, sums, early);
        } else if constexpr (EarlyBands<BM, BN, WM, WN>::ALL) {
            bands<BM, BN, WM, WN, SMEM>(p, t, N, acc, smem, wave, lane, early);
        } else if (p.chunks) {
            const bool part = N - t.n0 < BN && N % CH != 0;
            const auto go = [&](auto in) {
                constexpr int IN = decltype(in)::value;
                if (part) chunked<BM, BN, WM, WN, SMEM, IN, true>(p, t, N, acc, smem, wave, lane);
                else chunked<BM, BN, WM, WN, SMEM, IN, false>(p, t, N, acc, smem, wave, lane);
            };
            if (GRAD && p.codes) go(std::integral_constant<int, GRAD ? 2 : 0>{});
            else if (GRAD ? p.z != nullptr : p.res != nullptr) go(std::integral_constant<int, 1>{});
            else go(std::integral_constant<int, 0>{});
        } else {
            // Bands of 16 rows staged per wave, GB of them at a time, and read back as rows.
            // (The row loop stays rolled: its code, five activations long, would not fit the
            // instruction cache.)
            constexpr int LD = WTN + 4, NW = WM * WN;
            constexpr int GB = TM % 4 == 0 && NW * 64 * LD * 4 <= SMEM ? 4
                               : TM % 2 == 0 && NW * 32 * LD * 4 <= SMEM ? 2 : 1;
            static_assert(NW * GB * 16 * LD * 4 <= SMEM && WM * BN * 4 <= SMEM, "LDS");
            constexpr int CPR = WTN / CH, RPP = 64 / CPR;  // chunks per row, rows per pass
            constexpr int PASSES = GB * 16 / RPP;          // ... and group of bands
            static_assert(RPP <= 16, "a pass lies in one band group");
            float *const stg = (float *)smem + wave * GB * 16 * LD;
            const int r0 = lane / CPR, c = lane % CPR * CH, col = t.n0 + wn * WTN + c;
            const Flags fl(p);
            float bias[CH], sum[CH] = {};
            bias_of(p, col, N, bias);
            const int last = t.rows < (wm + 1) * WTM ? t.rows : (wm + 1) * WTM;
            int row = wm * WTM + r0;  // of the tile, this lane's in the next pass
            In next = load(p, t.row0 + row, col, N, row < last);
#pragma unroll
            for (int h = 0; h < TM / GB; ++h) {
#pragma unroll
                for (int i = 0; i < GB; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        *(v4f *)(stg + (i * 16 + l16) * LD + j * 16 + 4 * lq) = acc[h * GB + i][j];
                __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (int s = 0; s < PASSES; ++s) {
                    const In in = next;
                    const int at = row;
                    row += RPP;
                    next = load(p, t.row0 + row, col, N, row < last);
                    float f[CH];
#pragma unroll
                    for (int i = 0; i < CH; i += 4) {
                        const v4f v = *(const v4f *)(stg + (s * RPP + r0) * LD + c + i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[i + e] = v[e];
                    }
                    if (at < last) {
                        store(p, fl, t.row0 + at, col, N, bias, in, f);
                        if constexpr (GRAD) {
#pragma unroll
                            for (int e = 0; e < CH; ++e) sum[e] += f[e];
                        }
                    }
                }
                __builtin_amdgcn_s_waitcnt(0xC07F);
                __builtin_amdgcn_wave_barrier();
            }
            if (GRAD && p.sums) tile_sums<BM, BN, WM, WN>(p, t, N, sum, smem, wave, lane);
        }
    }

    // tile() of few passes, whose inputs are all there: bands of 16 rows staged per wave and read
    // back as rows.
    template <int BM, int BN, int WM, int WN, int SMEM, int TM, int TN>
    __device__ __forceinline__ static void bands(const Params &p, const RaggedTile &t, int N,
                                                 const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                                 int lane, const EarlyBands<BM, BN, WM, WN> &early) {
        using EB = EarlyBands<BM, BN, WM, WN>;
        constexpr int WTN = EB::WTN, LD = WTN + 4, RPP = EB::RPP, P = EB::P;
        constexpr int GB = WM * WN * TM * 16 * LD * 4 <= SMEM ? TM : TM / 2;  // bands staged at once
        static_assert(WM * WN * GB * 16 * LD * 4 <= SMEM && WM * BN * 4 <= SMEM, "LDS");
        const int wm = wave / WN, wn = wave % WN, l16 = lane & 15, lq = lane >> 4;
        const int r0 = lane / EB::CPR, c = lane % EB::CPR * CH, col = t.n0 + wn * WTN + c;
        float *const stg = (float *)smem + wave * GB * 16 * LD;
        const Flags fl(p);
        float sum[CH] = {};
#pragma unroll
        for (int i = 0; i < TM * P; ++i) {
            if (i % (GB * P) == 0) {
                __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses take effect in order)
#pragma unroll
                for (int b = 0; b < GB; ++b)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        *(v4f *)(stg + (b * 16 + l16) * LD + j * 16 + 4 * lq) = acc[i / P + b][j];
                __builtin_amdgcn_wave_barrier();
            }
            float f[CH];
#pragma unroll
            for (int k = 0; k < CH; k += 4) {
                const v4f v = *(const v4f *)(stg + (i % (GB * P) * RPP + r0) * LD + c + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[k + e] = v[e];
            }
            const int row = wm * TM * 16 + i * RPP + r0;
            if (row < t.rows) {
                store(p, fl, t.row0 + row, col, N, early.bias, early.in[i], f);
                if constexpr (GRAD) {
#pragma unroll
                    for (int e = 0; e < CH; ++e) sum[e] += f[e];
                }
            }
        }
        if (GRAD && p.sums) tile_sums<BM, BN, WM, WN>(p, t, N, sum, smem, wave, lane);
    }

    // Column sums of a tile from its lanes': lanes of the same columns, then the waves above each
    // other, in order.
    template <int BM, int BN, int WM, int WN>
    __device__ __forceinline__ static void tile_sums(const Params &p, const RaggedTile &t, int N,
                                                     float (&sum)[CH], uint8_t *smem, int wave,
                                                     int lane) {
        constexpr int WTN = BN / WN, CPR = WTN / CH;
        const int wm = wave / WN, wn = wave % WN;
#pragma unroll
        for (int d = CPR; d < 64; d <<= 1)
#pragma unroll
            for (int e = 0; e < CH; ++e) sum[e] += __shfl_xor(sum[e], d);
        __syncthreads();
        float *const red = (float *)smem;
        if (lane < CPR) {
#pragma unroll
            for (int e = 0; e < CH; ++e) red[wm * BN + wn * WTN + lane * CH + e] = sum[e];
        }
        __syncthreads();
        for (int j = threadIdx.x; j < BN; j += WM * WN * 64) {
            float s = red[j];
#pragma unroll
            for (int w = 1; w < WM; ++w) s += red[w * BN + j];
            put_sum<BM>(p, t, N, j, s);
        }
    }

    // tile() where every view has unit column stride, at any alignment: no branch
    // around any access, so that the wait for a band's inputs, which go out a band before it, is a
    // wait for them alone.  (Loads and stores share one counter: behind branches the compiler
    // waits for all of the stores too, every pass.)  One band is staged while the one before
    // it is worked on; the code of a band is there once, with a branch for its registers.
    // IN: the inputs, none, a matrix (the residual or bf16 pre-activations) or (2) a checkpoint.
    // PART: the matrix ends inside a chunk of this tile, whose elements go one by one.
    template <int BM, int BN, int WM, int WN, int SMEM, int IN, bool PART, int TM, int TN>
    __device__ __forceinline__ static void chunked(const Params &p, const RaggedTile &t, int N,
                                                   const v4f (&acc)[TM][TN], uint8_t *smem,
                                                   int wave, int lane) {
        constexpr int WTM = BM / WM, WTN = BN / WN, NW = WM * WN, LD = WTN + 4, ESZ = F32 ? 4 : 2;
        constexpr int CPR = WTN / CH, RPP = 64 / CPR, P = 16 / RPP;
        static_assert(NW * 2 * 16 * LD * 4 <= SMEM && WM * BN * 4 <= SMEM, "LDS");
        const int wm = wave / WN, wn = wave % WN, l16 = lane & 15, lq = lane >> 4;
        const int r0 = lane / CPR, c = lane % CPR * CH, cw = wn * WTN + c, col = t.n0 + cw;
        const int cols = N - t.n0 < BN ? N - t.n0 : BN, row = wm * WTM + r0;
        const bool in_c = cw < cols, in_b = cw < ((cols + 31) & ~31);
        const Flags fl(p);
        const int64_t row0 = t.row0;
        const int64_t ldc = (p.rsc > N ? p.rsc : N) * ESZ;  // (one row: any stride)
        Rows rc((uint8_t *)p.c + row0 * ldc + t.n0 * ESZ, ldc, t.rows, cols * ESZ, row, cw * ESZ, in_c, RPP);
        // inputs: the residual, or the pre-activations
        constexpr int ISZ = GRAD ? 2 : ESZ;
        const void *const ip = GRAD ? (const void *)p.z : p.res;
        const int64_t ldi = (!GRAD ? p.rsr : p.rsz > N ? p.rsz : N) * ISZ;
        Rows ri((const uint8_t *)ip + row0 * ldi + t.n0 * ISZ, ldi, t.rows, cols * ISZ, row, cw * ISZ, in_c, RPP);
        const int64_t ldz = (p.rsz > N ? p.rsz : N) * 2;
        Rows rz((uint8_t *)p.z + row0 * ldz + t.n0 * 2, ldz, t.rows, cols * 2, row, cw * 2, in_c, RPP);
        Rows rq(p.codes + row0 * p.ld + t.n0, p.ld, t.rows, (cols + 31) & ~31, row, cw, in_b, RPP);
        Rows rs(p.scales + row0 * p.lds + (t.n0 >> 5), p.lds, t.rows, (cols + 31) >> 5, row, cw >> 5,
                in_b && (GRAD || (cw & 31) == 0), RPP);
        float bias[CH], sum[CH] = {};
        bias_of(p, col, N, bias);

        struct Raw : In {
            uint32_t raw[IN == 1 && PART ? CH : 1];
        };
        auto load_in = [&](Raw &in) {
            if constexpr (IN == 2) {
                if constexpr (CH == 8) {
                    const v2u w = __builtin_amdgcn_raw_buffer_load_b64(rq.r, rq.at, 0, 0);
                    in.v[0] = w[0];
                    in.v[1] = w[1];
                } else {
                    in.v[0] = __builtin_amdgcn_raw_buffer_load_b32(rq.r, rq.at, 0, 0);
                }
                in.byte = (int)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs.r, rs.at, 0, 0);
                rq.at += rq.step;
                rs.at += rs.step;
            } else if constexpr (IN == 1 && PART) {
                ri.template load<CH, ISZ>(in.raw, N - col);
            } else if constexpr (IN == 1) {
                if constexpr (CH * ISZ == 16) {
                    in.v = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(ri.r, ri.at, 0, 0));
                } else {
                    const v2u w = __builtin_amdgcn_raw_buffer_load_b64(ri.r, ri.at, 0, 0);
                    in.v[0] = w[0];
                    in.v[1] = w[1];
                }
                ri.at += ri.step;
            }
        };
        float *const stg = (float *)smem + wave * 2 * 16 * LD;
        auto stage = [&](int h) {  // band h of 1 .. TM - 1
            float *const d = stg + (h & 1) * 16 * LD + l16 * LD + 4 * lq;
#pragma unroll
            for (int i = 1; i < TM; ++i) {
                // (opaque, so that the branches stay apart: merged they would index the
                // accumulators through scratch memory)
                int k = h;
                asm volatile("" : "+s"(k));
                if (k == i) {
#pragma unroll
                    for (int j = 0; j < TN; ++j) *(v4f *)(d + j * 16) = acc[i][j];
                }
            }
        };
        constexpr int D = TM % kAhead == 0 ? kAhead : TM;
        Raw next[D][P];
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int s = 0; s < P; ++s) load_in(next[d][s]);
#pragma unroll
        for (int j = 0; j < TN; ++j) *(v4f *)(stg + l16 * LD + 4 * lq + j * 16) = acc[0][j];
        int at_row = row;
#pragma unroll 1
        for (int h0 = 0; h0 < TM; h0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int h = h0 + d;
                Raw in[P];
#pragma unroll
                for (int s = 0; s < P; ++s) in[s] = next[d][s];
                // (past the wave's last band: rows of the next wave or none, not used)
#pragma unroll
                for (int s = 0; s < P; ++s) load_in(next[d][s]);
                __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses take effect in order)
                stage(h + 1);
                const float *const src = stg + (h & 1) * 16 * LD + r0 * LD + c;
#pragma unroll
                for (int s = 0; s < P; ++s) {
                    float f[CH];
#pragma unroll
                    for (int i = 0; i < CH; i += 4) {
                        const v4f v = *(const v4f *)(src + s * RPP * LD + i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[i + e] = v[e];
                    }
                    if constexpr (IN == 1 && PART) in[s].v = packed<CH, ISZ>(in[s].raw);
                    if constexpr (GRAD) {
                        grad_map(p, p.alpha, IN, in[s], f);
                        // (rows that are not there: no zeros where a column of B is infinite)
#pragma unroll
                        for (int e = 0; e < CH; ++e) sum[e] += at_row < t.rows ? f[e] : 0.0f;
                        at_row += RPP;
                    } else {
#pragma unroll
                        for (int e = 0; e < CH; ++e) f[e] = __builtin_fmaf(p.alpha, f[e], bias[e]);
                        if (p.codes) {
                            v2u w;
                            const int byte = quantize(f, w);
                            if constexpr (CH == 8) __builtin_amdgcn_raw_buffer_store_b64(w, rq.r, rq.at, 0, 0);
                            else __builtin_amdgcn_raw_buffer_store_b32(w[0], rq.r, rq.at, 0, 0);
                            __builtin_amdgcn_raw_buffer_store_b8((uint8_t)byte, rs.r, rs.at, 0, 0);
                            rq.at += rq.step;
                            rs.at += rs.step;
                        } else if (p.z) {
                            put<false, PART>(rz, fl.nt_z, N - col, f);
                        }
                        act_map(p, IN == 1, in[s], f);
                    }
                    put<F32, PART>(rc, fl.nt_c, N - col, f);
                }
            }
        }
        if (GRAD && p.sums) tile_sums<BM, BN, WM, WN>(p, t, N, sum, smem, wave, lane);
    }

    // A chunk, rounded once, to its place in the next pass.
    template <bool W, bool PART>
    __device__ __forceinline__ static void put(Rows &r, bool nt, int cols, const float (&f)[CH]) {
        v4u w = {};
        if constexpr (W) {
#pragma unroll
            for (int e = 0; e < CH; ++e) w[e % 4] = __float_as_uint(f[e]);
        } else {
#pragma unroll
            for (int e = 0; e < CH / 2; ++e) w[e] = bf16x2_rne(f[2 * e], f[2 * e + 1]);
        }
        r.template store<CH, W ? 4 : 2, PART>(w, cols, nt);
    }
};

// ---------------------------------------------------------------- launch

// f(the tile of a linear layer's product): that of forward_tile, but for products of which 16 x 32
// pieces are more than a CU each and 32 x 32 pieces are not: those take 32 x 32, K split over four
// waves.  Graph-timed with rotating weights, us against the other rule's: 64x14336x4096 38.5 / 56.0,
// 64x4096x4096 12.6 / 18.0, 128x2048x2048 6.2 / 8.0, 100x1000x1504 4.7 / 6.0, 333x512x512 3.8 / 4.4
// (n-contiguous weights 58.8 / 66.8, 19.1 / 21.4, 7.1 / 8.0, 5.1 / 6.0, 4.0 / 4.5).
template <bool BT, typename F>
static auto linear_tile(const RaggedArgs &g, F f) {
    if (g.any_align) return any_align_tile(g, f);
    const int64_t cols = ((int64_t)g.N + 31) / 32;
    if (((int64_t)g.M + 15) / 16 * cols > g.cus && ((int64_t)g.M + 31) / 32 * cols <= g.cus &&
        g.K >= 256)
        return f(WaveTile<32, 32, 4, 3>{});
    return forward_tile<false, BT>(g, f);
}

template <bool BT, EpiKind E, bool GRAD>
static hipError_t linear_go(const RaggedArgs &g, const LinearParams &p, hipStream_t stream) {
    return linear_tile<BT>(g, [&](auto t) {
        return ragged_go<false, false, BT, LinearOut<E, GRAD>, decltype(t)>(g, p, stream);
    });
}

// Whether a view has unit column stride, at any alignment, and rows in reach of a tile's 32-bit
// offsets (LinearOut::chunked, whose PART takes chunks that the matrix cuts).
inline bool chunk_rows(int64_t rs, int64_t cs, int64_t M, int64_t size) {
    return cs == 1 && (M <= 1 || rs * size <= kMaxTileRowBytes);
}

template <bool GRAD>
static hipError_t linear_launch(const RaggedArgs &g, RaggedB bl, EpiKind kind, LinearParams p,
                                hipStream_t stream) {
    const bool cols = bl == RaggedB::Cols;
    const int64_t size = kind == EpiKind::F32 ? 4 : 2;
    p.chunks = chunk_rows(p.rsc, p.csc, g.M, size) &&
               (!p.res || chunk_rows(p.rsr, p.csr, g.M, size)) &&
               (!p.z || (chunk_rows(p.rsz, p.csz, g.M, 2) && (g.M <= 1 || p.rsz >= g.N))) &&
               (!p.codes || (p.ld <= kMaxTileRowBytes && p.lds <= kMaxTileRowBytes)) &&
               (int64_t)g.N * size <= kMaxTileRowBytes;
    if (g.M == 1) p.rsc = p.rsr = p.rsz = 0;  // (never used)
    if (kind == EpiKind::BF16)
        return cols ? linear_go<true, EpiKind::BF16, GRAD>(g, p, stream)
                    : linear_go<false, EpiKind::BF16, GRAD>(g, p, stream);
    if (kind == EpiKind::F32)
        return cols ? linear_go<true, EpiKind::F32, GRAD>(g, p, stream)
                    : linear_go<false, EpiKind::F32, GRAD>(g, p, stream);
    return hipErrorInvalidValue;
}

}  // namespace gk
