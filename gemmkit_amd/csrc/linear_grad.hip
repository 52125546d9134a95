// linear_grad.hip -- the input gradients of linear layers through the activation before
// them (linear.h), the activation's gradient alone, and the sums of column sums.
#include <algorithm>

#include "linear.h"

namespace gk {

hipError_t launch_linear_grad(const RaggedArgs &g, RaggedB bl, EpiKind kind, const LinearParams &p,
                              hipStream_t stream) {
    return linear_launch<true>(g, bl, kind, p, stream);
}

int linear_unit(const RaggedArgs &g, RaggedB bl) { return sum_unit(grouped_plan(g, bl).bm); }

// ---------------------------------------------------------------- activation gradient

// C = A * act'(Z), a workgroup per 256 >> ty chunk columns of 8 and `unit` rows, 1 << ty rows
// at a time; column sums of its rows before rounding to one row of p.sums.

// The workgroup's column sums from its threads': column j of the strip, its rows' sums in order.
__device__ __forceinline__ void strip_sums(const LinearParams &p, int N, int tx, int ty, float *red,
                                           const float (&sum)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = sum[e];
    __syncthreads();
    const int width = 8 << tx, base = (int)blockIdx.x * width;
    for (int j = threadIdx.x; j < width; j += 256) {
        float s = 0.0f;
        for (int y = 0; y < 1 << ty; ++y) s += red[(y << tx) * 8 + j];
        if (base + j < N) p.sums[(int64_t)blockIdx.y * N + base + j] = s;
    }
}

// Every view of unit column stride and whole chunks (LinearOut::chunked): no branch around any
// access, and the next U rows' inputs go out before this one's stores.
// IN: pre-activations, none, bf16, or (2) a checkpoint.
template <InType T, int IN>
__global__ __launch_bounds__(256) void act_grad_rows_kernel(const LinearParams p, int64_t M, int N,
                                                            int unit, int ty) {
    constexpr bool F32 = T == InType::F32;
    constexpr int U = 2, SZ = F32 ? 4 : 2;
    __shared__ float red[256 * 8];
    const int tx = 8 - ty, cx = threadIdx.x & ((1 << tx) - 1), ry = threadIdx.x >> tx;
    const int width = 8 << tx, n0 = (int)blockIdx.x * width, c = cx * 8;
    const int cols = N - n0 < width ? N - n0 : width;
    const int64_t row0 = (int64_t)blockIdx.y * unit;
    const int rows = M - row0 < unit ? (int)(M - row0) : unit;
    const bool in = c < cols, nt = row_lines(p.c, p.rsc * 2);
    const int rpp = 1 << ty;
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
    };
    auto load = [&](In &i) {
        i.a[0] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(ra.r, ra.at, 0, 0));
        if constexpr (F32)
            i.a[1] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(ra.r, ra.at + 16, 0, 0));
        ra.at += ra.step;
        if constexpr (IN == 2) {
            const v2u w = __builtin_amdgcn_raw_buffer_load_b64(rq.r, rq.at, 0, 0);
            i.z[0] = w[0];
            i.z[1] = w[1];
            i.byte = (int)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs.r, rs.at, 0, 0);
            rq.at += rq.step;
            rs.at += rs.step;
        } else if constexpr (IN == 1) {
            i.z = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rz.r, rz.at, 0, 0));
            rz.at += rz.step;
        }
    };
    float sum[8] = {};
    In next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(next[u]);
#pragma unroll 1
    for (int r = 0; r < rows; r += U << ty) {
        In i[U];
#pragma unroll
        for (int u = 0; u < U; ++u) i[u] = next[u];
#pragma unroll
        for (int u = 0; u < U; ++u) load(next[u]);  // (past the end: zeros)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[8];
            if constexpr (F32) {
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
            if (nt) __builtin_amdgcn_raw_buffer_store_b128(w, rc.r, rc.at, 0, 2);
            else __builtin_amdgcn_raw_buffer_store_b128(w, rc.r, rc.at, 0, 0);
            rc.at += rc.step;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
    }
    if (p.sums) strip_sums(p, N, tx, ty, red, sum);
}

// Views of any strides.
template <InType T>
__global__ __launch_bounds__(256) void act_grad_kernel(const LinearParams p, int64_t M, int N,
                                                       int unit, int ty) {
    constexpr bool F32 = T == InType::F32;
    constexpr int U = 4;  // rows whose loads are in flight together
    __shared__ float red[256 * 8];
    const int tx = 8 - ty, cx = threadIdx.x & ((1 << tx) - 1), ry = threadIdx.x >> tx;
    const int col = ((int)blockIdx.x << tx | cx) * 8, cols = N - col;
    const int64_t first = (int64_t)blockIdx.y * unit;
    const int64_t end = first + unit < M ? first + unit : M;
    const bool nt = row_lines(p.c, p.rsc * 2);
    float sum[8] = {};
    if (cols > 0) {
        for (int64_t r = first + ry; r < end; r += (int64_t)U << ty) {
            v4u a[U][2], z[U];
            int byte[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + ((int64_t)u << ty);
                a[u][0] = a[u][1] = z[u] = v4u{};
                byte[u] = 0;
                if (row >= end) continue;
                if constexpr (F32) {
                    a[u][0] = read_raw<true, 4>(p.res, row * p.rsr + col * p.csr, p.csr, cols);
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
                const int64_t row = r + ((int64_t)u << ty);
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
    if (p.sums) strip_sums(p, N, tx, ty, red, sum);
}

// Rows that share a thread's columns: 64 chunk columns (a KiB of bf16 in a row) where the matrix
// has them.
static int act_grad_ty(int64_t n) {
    int tx = 6;
    while (tx > 0 && ((int64_t)8 << (tx - 1)) >= n) --tx;
    return 8 - tx;
}

int act_grad_unit(int64_t m, int64_t n, int cus) {
    const int ty = act_grad_ty(n);
    const int64_t strips = (n + (2048 >> ty) - 1) / (2048 >> ty);
    // about eight workgroups per CU, of at least one row per thread
    const int64_t parts = std::max<int64_t>(8 * (int64_t)cus / strips, 1), rows = (m + parts - 1) / parts;
    int64_t unit = (rows + (1 << ty) - 1) >> ty << ty;
    unit = std::max<int64_t>(unit, 1 << ty);
    return (int)std::max<int64_t>(unit, (m + 65534) / 65535);
}

template <InType T>
static void act_grad_go(const LinearParams &p, int64_t m, int64_t n, int unit, int ty, dim3 grid,
                        hipStream_t stream) {
    // (32-bit offsets: the rows of a workgroup)
    const int64_t most = (int64_t)kMaxRecords / (unit + (4 << ty));
    const auto rows = [&](const void *q, int64_t rs, int64_t cs, int64_t size) {
        return cs == 1 && (uintptr_t)q % 4 == 0 &&
               (m <= 1 || (rs * size % 4 == 0 && rs >= n && rs * size <= most));
    };
    const int64_t size = (int64_t)in_size(T);
    const bool chunks = n % 8 == 0 && n * 4 <= most && rows(p.c, p.rsc, p.csc, 2) &&
                        rows(p.res, p.rsr, p.csr, size) && (!p.z || rows(p.z, p.rsz, p.csz, 2)) &&
                        (!p.codes || (p.ld <= most && p.lds <= most));
    LinearParams q = p;
    if (m == 1) q.rsc = q.rsr = q.rsz = 0;  // (never used)
    if (!chunks)
        hipLaunchKernelGGL((act_grad_kernel<T>), grid, dim3(256), 0, stream, q, m, (int)n, unit, ty);
    else if (p.codes)
        hipLaunchKernelGGL((act_grad_rows_kernel<T, 2>), grid, dim3(256), 0, stream, q, m, (int)n, unit, ty);
    else if (p.z)
        hipLaunchKernelGGL((act_grad_rows_kernel<T, 1>), grid, dim3(256), 0, stream, q, m, (int)n, unit, ty);
    else
        hipLaunchKernelGGL((act_grad_rows_kernel<T, 0>), grid, dim3(256), 0, stream, q, m, (int)n, unit, ty);
}

hipError_t launch_act_grad(InType in, int64_t m, int64_t n, int cus, const LinearParams &p,
                           hipStream_t stream) {
    const int ty = act_grad_ty(n), unit = act_grad_unit(m, n, cus);
    const dim3 grid((uint32_t)((n + (2048 >> ty) - 1) / (2048 >> ty)), (uint32_t)((m + unit - 1) / unit));
    if (in == InType::BF16) act_grad_go<InType::BF16>(p, m, n, unit, ty, grid, stream);
    else act_grad_go<InType::F32>(p, m, n, unit, ty, grid, stream);
    return hipGetLastError();
}

// ---------------------------------------------------------------- column sums

// 32 columns a workgroup; eight lanes of rows each add every eighth row, then the eight.
__global__ __launch_bounds__(256) void col_sums_kernel(const float *part, int64_t rows, int64_t n,
                                                       float *out) {
    __shared__ float red[256];
    const int c = threadIdx.x & 31, l = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    float s = 0.0f;
    if (col < n) {
#pragma unroll 8
        for (int64_t r = l; r < rows; r += 8) s += part[r * n + col];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (l == 0 && col < n) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += red[i * 32 + c];
        out[col] = s;
    }
}

hipError_t launch_col_sums(const float *part, int64_t rows, int64_t n, float *out, hipStream_t stream) {
    hipLaunchKernelGGL(col_sums_kernel, dim3((uint32_t)((n + 31) / 32)), dim3(256), 0, stream, part,
                       rows, n, out);
    return hipGetLastError();
}

}  // namespace gk
