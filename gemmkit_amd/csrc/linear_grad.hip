// linear_grad.hip -- the input gradients of linear layers through the activation before
// them (linear.h), the activation's gradient alone, and the sums of column sums.
#include <algorithm>

#include "linear.h"

namespace gk {

hipError_t launch_linear_grad(const RaggedArgs &g, RaggedB bl, EpiKind kind, const LinearParams &p,
                              hipStream_t stream) {
    return linear_launch<true>(g, bl, kind, p, stream);
}

int linear_unit(const RaggedArgs &g, RaggedB bl) {
    const auto unit = [](auto t) { return sum_unit(decltype(t)::BM); };
    return bl == RaggedB::Cols ? linear_tile<true>(g, unit) : linear_tile<false>(g, unit);
}

// ---------------------------------------------------------------- activation gradient

// C = A * act'(Z), a workgroup per strip of 1 << tx chunk columns of 8 and `unit` rows, as many rows at
// a time as it has threads for; column sums of its rows before rounding to one row of p.sums.
constexpr int kStripSums = 4 * 512;  // floats: four waves of 64 chunk columns, or 16 of four
constexpr int kStripTx = 2;  // narrow strips of aligned rows
constexpr int64_t kStripElems = (int64_t)3 << 20;  // ... of others, at most

// The workgroup's column sums from its threads': a wave's rows, then the waves, in order.
template <int THREADS>
__device__ __forceinline__ void strip_sums(const LinearParams &p, int strip, int N, int tx, float *red,
                                           float (&sum)[8]) {
    for (int d = 1 << tx; d < 64; d <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], d);
    const int width = 8 << tx, base = strip * width, lane = threadIdx.x & 63;
    if (lane < 1 << tx) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[(threadIdx.x >> 6) * width + lane * 8 + e] = sum[e];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < width; j += THREADS) {
        float s = red[j];
        for (int w = 1; w < THREADS / 64; ++w) s += red[w * width + j];
        if (base + j < N) p.sums[(int64_t)blockIdx.y * N + base + j] = s;
    }
}

// Views of unit column stride (LinearOut::chunked): no branch around any access, and the next U
// rows' inputs go out before this one's stores.
// IN: pre-activations, none, bf16, or (2) a checkpoint.  PART: the matrix ends inside a chunk.
// ONCE: G nontemporally.
template <InType T, int IN, bool PART, bool ONCE, int THREADS>
__device__ __forceinline__ void act_grad_rows(const LinearParams &p, int strip, int64_t M, int N,
                                              int unit, int tx, float *red) {
    constexpr bool F32 = T == InType::F32;
    constexpr int U = 2, SZ = F32 ? 4 : 2, AUX = ONCE ? 2 : 0;
    const int cx = threadIdx.x & ((1 << tx) - 1), ry = threadIdx.x >> tx;
    const int width = 8 << tx, n0 = strip * width, c = cx * 8;
    const int cols = N - n0 < width ? N - n0 : width;
    const int64_t row0 = (int64_t)blockIdx.y * unit;
    const int rows = M - row0 < unit ? (int)(M - row0) : unit;
    const bool in = c < cols, nt = row_lines(p.c, p.rsc * 2);
    const int rpp = THREADS >> tx;
    const int64_t ldc = (p.rsc > N ? p.rsc : N) * 2, ldz = (p.rsz > N ? p.rsz : N) * 2;
    const int64_t lda = (p.rsr > N ? p.rsr : N) * SZ;
    Rows rc((uint8_t *)p.c + row0 * ldc + n0 * 2, ldc, rows, cols * 2, ry, c * 2, in, rpp);
    Rows ra((const uint8_t *)p.res + row0 * lda + n0 * SZ, lda, rows, cols * SZ, ry, c * SZ, in, rpp);
    Rows rz((const uint8_t *)p.z + row0 * ldz + n0 * 2, ldz, rows, cols * 2, ry, c * 2, in, rpp);
    Rows rq(p.codes + row0 * p.ld + n0, p.ld, rows, (cols + 31) & ~31, ry, c, in, rpp);
    Rows rs(p.scales + row0 * p.lds + (n0 >> 5), p.lds, rows, (cols + 31) >> 5, ry, c >> 5, in, rpp);
    struct In {
        v4u a[F32 ? 2 : 1], z;
        int byte;
        uint32_t ra[PART ? 8 : 1], rz[PART && IN == 1 ? 8 : 1];
    };
    const int left = N - n0 - c;
    auto load = [&](In &i) {
        if constexpr (PART) {
            ra.template load<8, SZ>(i.ra, left);
            if constexpr (IN == 1) rz.template load<8, 2>(i.rz, left);
        }
        if constexpr (!PART) {
            i.a[0] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(ra.r, ra.at, 0, AUX));
            if constexpr (F32)
                i.a[1] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(ra.r, ra.at + 16, 0, AUX));
            ra.at += ra.step;
            if constexpr (IN == 1) {
                i.z = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rz.r, rz.at, 0, 0));
                rz.at += rz.step;
            }
        }
        if constexpr (IN == 2) {
            const v2u w = __builtin_amdgcn_raw_buffer_load_b64(rq.r, rq.at, 0, 0);
            i.z[0] = w[0];
            i.z[1] = w[1];
            i.byte = (int)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs.r, rs.at, 0, 0);
            rq.at += rq.step;
            rs.at += rs.step;
        }
    };
    float sum[8] = {};
    In next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(next[u]);
#pragma unroll 1
    for (int r = 0; r < rows; r += U * rpp) {
        In i[U];
#pragma unroll
        for (int u = 0; u < U; ++u) i[u] = next[u];
#pragma unroll
        for (int u = 0; u < U; ++u) load(next[u]);  // (past the end: zeros)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[8];
            if constexpr (PART) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(F32 ? i[u].ra[e] : i[u].ra[e] << 16);
                if constexpr (IN == 1) i[u].z = packed<8, 2>(i[u].rz);
            } else if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(i[u].a[F32 ? e / 4 : 0][e % 4]);
            } else {
                widen<false, 8>(i[u].a[0], f);
            }
            if constexpr (IN != 0) {
                float z[8];
                if constexpr (IN == 2) {
                    const float step = mxint8_step(i[u].byte);
                    mxint8_values4(i[u].z[0], step, z);
                    mxint8_values4(i[u].z[1], step, z + 4);
                } else {
                    widen<false, 8>(i[u].z, z);
                }
                act_scale(f, z, p.act, p.slope);
            }
            v4u w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = bf16x2_rne(f[2 * e], f[2 * e + 1]);
            rc.template store<8, 2, PART>(w, left, nt);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
    }
    if (p.sums) strip_sums<THREADS>(p, strip, N, tx, red, sum);
}

// A strip of any strides and width.
template <InType T, int THREADS>
__device__ __forceinline__ void act_grad_any(const LinearParams &p, int strip, int64_t M, int N,
                                             int unit, int tx, float *red) {
    constexpr bool F32 = T == InType::F32;
    constexpr int U = 2;  // rows whose loads are in flight together
    const int cx = threadIdx.x & ((1 << tx) - 1), ry = threadIdx.x >> tx, rpp = THREADS >> tx;
    const int col = (strip << tx | cx) * 8, cols = N - col;
    const int64_t first = (int64_t)blockIdx.y * unit;
    const int64_t end = first + unit < M ? first + unit : M;
    const bool nt = row_lines(p.c, p.rsc * 2);
    float sum[8] = {};
    if (cols > 0) {
        for (int64_t r = first + ry; r < end; r += (int64_t)U * rpp) {
            v4u a[U][2], z[U];
            int byte[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + (int64_t)u * rpp;
                a[u][0] = a[u][1] = z[u] = v4u{};
                byte[u] = 0;
                if (row >= end) continue;
                if constexpr (F32) {
                    a[u][0] = read_raw<true, 4>(p.res, row * p.rsr + col * p.csr, p.csr, cols);
                    if (cols > 4)
                        a[u][1] = read_raw<true, 4>(p.res, row * p.rsr + (col + 4) * p.csr, p.csr, cols - 4);
                } else {
                    a[u][0] = read_raw<false, 8>(p.res, row * p.rsr + col * p.csr, p.csr, cols);
                }
                if (p.codes) {
                    const v2u w = *(const v2u *)(p.codes + row * p.ld + col);
                    z[u][0] = w[0];
                    z[u][1] = w[1];
                    byte[u] = p.scales[row * p.lds + (col >> 5)];
                } else if (p.z) {
                    z[u] = read_raw<false, 8>(p.z, row * p.rsz + col * p.csz, p.csz, cols);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + (int64_t)u * rpp;
                if (row >= end) break;
                float f[8];
                if constexpr (F32) {
                    float lo[4], hi[4];
                    widen<true, 4>(a[u][0], lo);
                    widen<true, 4>(a[u][1], hi);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f[e] = lo[e];
                        f[4 + e] = hi[e];
                    }
                } else {
                    widen<false, 8>(a[u][0], f);
                }
                if (p.act != kActNone) {
                    float v[8];
                    if (p.codes) {
                        const float step = mxint8_step(byte[u]);
                        mxint8_values4(z[u][0], step, v);
                        mxint8_values4(z[u][1], step, v + 4);
                    } else {
                        widen<false, 8>(z[u], v);
                    }
                    act_scale(f, v, p.act, p.slope);
                }
                write_row<false, 8>(p.c, row * p.rsc + col * p.csc, p.csc, cols, nt, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += f[e];
            }
        }
    }
    if (p.sums) strip_sums<THREADS>(p, strip, N, tx, red, sum);
}

// IN 0..2: act_grad_rows; 3: views of any strides.
template <InType T, int IN, bool ONCE, int THREADS>
__global__ __launch_bounds__(THREADS) void act_grad_kernel(const LinearParams p, int64_t M, int N,
                                                           int unit, int tx) {
    __shared__ float red[kStripSums];
    int strip = (int)blockIdx.x;
    if (tx == kStripTx && gridDim.y == 1) {  // neighbours, which share lines, on one XCD
        const int x = strip % 8, per = (int)gridDim.x / 8, more = (int)gridDim.x % 8;
        strip = x * per + (x < more ? x : more) + strip / 8;
    }
    if constexpr (IN == 3) {
        act_grad_any<T, THREADS>(p, strip, M, N, unit, tx, red);
    } else {
        const bool part = N % 8 != 0 && N - (strip << (3 + tx)) < 8 << tx;
        if (part) act_grad_rows<T, IN, true, ONCE, THREADS>(p, strip, M, N, unit, tx, red);
        else act_grad_rows<T, IN, false, ONCE, THREADS>(p, strip, M, N, unit, tx, red);
    }
}

// Whether every row of the views starts at 16 bytes.
static bool act_grad_aligned(InType in, int64_t m, const LinearParams &p) {
    const auto rows = [&](const void *q, int64_t rs, int64_t cs, int64_t size) {
        return cs == 1 && (((uint64_t)q | (m > 1 ? (uint64_t)(rs * size) : 0)) & 15) == 0;
    };
    return rows(p.c, p.rsc, p.csc, 2) && rows(p.res, p.rsr, p.csr, (int64_t)in_size(in)) &&
           (!p.z || rows(p.z, p.rsz, p.csz, 2));
}

// A workgroup's part.  Strips of 64 chunk columns (a KiB of bf16 in a row) where the matrix has
// them, rows for about eight workgroups per CU, at least two per thread.  Column sums of few rows:
// narrow strips of all rows, which need no second launch.  Aligned rows up to 1024, four chunk
// columns (calls, us, against two launches: bf16 512 x 8192 9.4 / 12.0, 1024 x 1024 9.6 / 14.3, 1024 x 8192
// 10.9 / 14.9; 2048 x 4096 14.3 / 14.6, 2048 x 8192 18.8 / 19.2).  Others are bound by their addresses on
// the few CUs of narrow strips, and from about 3 Mi elements on by the cache lines that strips of two
// chunk columns share: up to 512 rows (calls: 333 x 1501 9.0 / 13.5, 256 x 8001 10.3 / 14.5, 512 x 4001
// 10.4 / 14.3; 256 x 16001 18.8 / 14.4, 512 x 8001 17.5 / 15.6, f32 18.8 / 17.7, 512 x 65536 167 / 39;
// more rows: f32 1003 x 777 12.8 / 12.1 to 16, its kernels 12.8 / 10.1).
struct ActGradShape {
    int tx, unit, threads;
};
static ActGradShape act_grad_shape(InType in, int64_t m, int64_t n, int cus, const LinearParams &p,
                                   bool sums) {
    int tx = 6;
    while (tx > 0 && ((int64_t)8 << (tx - 1)) >= n) --tx;
    const int rpp = 256 >> tx;
    const int64_t strips = (n + (8 << tx) - 1) / (8 << tx);
    const int64_t parts = std::max<int64_t>(8 * (int64_t)cus / strips, 1), rows = (m + parts - 1) / parts;
    int64_t unit = (rows + rpp - 1) / rpp * rpp;
    unit = std::max<int64_t>(unit, 2 * rpp);
    unit = std::max<int64_t>(unit, (m + 65534) / 65535);
    if (sums && m > unit) {
        if (m <= 1024 && m * n * (int64_t)in_size(in) < kOnceBytes && act_grad_aligned(in, m, p))
            return {kStripTx, (int)m, m <= 256 ? 256 : 1024};
        if (m <= 512 && m * n <= kStripElems) return {1, (int)m, 256};
    }
    return {tx, (int)unit, 256};
}

int act_grad_unit(InType in, int64_t m, int64_t n, int cus, const LinearParams &p) {
    return act_grad_shape(in, m, n, cus, p, true).unit;
}

template <InType T>
static void act_grad_go(const LinearParams &p, int64_t m, int64_t n, const ActGradShape &shape,
                        hipStream_t stream) {
    // (32-bit offsets: the rows of a workgroup)
    const int tx = shape.tx, unit = shape.unit, threads = shape.threads;
    const dim3 grid((uint32_t)((n + (8 << tx) - 1) / (8 << tx)), (uint32_t)((m + unit - 1) / unit));
    const int64_t most = (int64_t)kMaxRecords / (unit + 4 * (threads >> tx));
    const auto rows = [&](int64_t rs, int64_t cs, int64_t size) {
        return cs == 1 && (m <= 1 || (rs >= n && rs * size <= most));
    };
    const bool chunks = n * 4 <= most && rows(p.rsc, p.csc, 2) &&
                        rows(p.rsr, p.csr, (int64_t)in_size(T)) && (!p.z || rows(p.rsz, p.csz, 2)) &&
                        (!p.codes || (p.ld <= most && p.lds <= most));
    LinearParams q = p;
    if (m == 1) q.rsc = q.rsr = q.rsz = 0;  // (never used)
    const auto go = [&](auto in, auto once) {
        constexpr int IN = decltype(in)::value;
        constexpr bool ONCE = decltype(once)::value;
        if (threads == 1024)
            hipLaunchKernelGGL((act_grad_kernel<T, IN, false, 1024>), grid, dim3(1024), 0, stream, q, m,
                               (int)n, unit, tx);
        else
            hipLaunchKernelGGL((act_grad_kernel<T, IN, ONCE, 256>), grid, dim3(256), 0, stream, q, m,
                               (int)n, unit, tx);
    };
    // (kernels, us, plain loads of G / nontemporal ones: bf16 8192 x 8192 70.4 / 65.1, 4096 x 8192
    // 37.6 / 36.9, 1024 x 8192 12.0 / 12.6; f32 4096 x 8192 54.4 / 49.3, 1024 x 8192 13.8 / 15.2; the
    // pre-activations nontemporally too 69.2 for the first)
    const bool once = m * n * (int64_t)in_size(T) >= kOnceBytes;
    const auto either = [&](auto in) {
        if (once) go(in, std::true_type{});
        else go(in, std::false_type{});
    };
    if (!chunks) go(std::integral_constant<int, 3>{}, std::false_type{});
    else if (p.codes) either(std::integral_constant<int, 2>{});
    else if (p.z) either(std::integral_constant<int, 1>{});
    else either(std::integral_constant<int, 0>{});
}

hipError_t launch_act_grad(InType in, int64_t m, int64_t n, int cus, const LinearParams &p,
                           hipStream_t stream) {
    const ActGradShape shape = act_grad_shape(in, m, n, cus, p, p.sums != nullptr);
    if (in == InType::BF16) act_grad_go<InType::BF16>(p, m, n, shape, stream);
    else act_grad_go<InType::F32>(p, m, n, shape, stream);
    return hipGetLastError();
}

// ---------------------------------------------------------------- column sums

// 16 columns a workgroup; sixteen lanes of rows each add every sixteenth row, then the sixteen.
__global__ __launch_bounds__(256) void col_sums_kernel(const float *part, int64_t rows, int64_t n,
                                                       float *out) {
    __shared__ float red[256];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4;
    const int64_t col = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16 + c;
    float s = 0.0f;
    if (col < n) {
#pragma unroll 8
        for (int64_t r = l; r < rows; r += 16) s += part[r * n + col];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (l == 0 && col < n) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i * 16 + c];
        out[col] = s;
    }
}

hipError_t launch_col_sums(const float *part, int64_t rows, int64_t n, float *out, hipStream_t stream) {
    // (from 2^28 columns on one row of workgroups would have more threads than 32 bits count)
    hipLaunchKernelGGL(col_sums_kernel, ragged_grid((n + 15) / 16), dim3(256), 0, stream, part, rows, n,
                       out);
    return hipGetLastError();
}

}  // namespace gk
