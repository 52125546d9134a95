#pragma once
// ragged.h -- products of ragged groups on the 16x16 matrix-core instructions.
//
// One workgroup computes a BM x BN tile of one group's product.  K advances in stages of
// 128 bytes per operand row (64 bf16, 256 e2m1 codes) through a ring of NS LDS slots filled
// by direct-to-LDS loads; out-of-range rows and K tails read zeros by the buffer
// resources' range check, as in mma_kernel.h.
//
// Operand layouts in memory and in a stage:
//   k-contiguous   W rows of 128 bytes, chunk c (16 bytes) of row r in slot c ^ swz(r):
//                  a fragment is one 16-byte read per lane.
//   transposed     (bf16) the contraction index is the slow one: 64 rows of W elements.
//                  ds_read_b64_tr_b16 gives lane l of a 16-lane group element l%16 of four
//                  consecutive rows, of which the group's lanes read 8 bytes each; two of
//                  them make the fragment (rows 8*(l/16) .. +7) that the k-contiguous read
//                  gives.  So weights stored input-major, and both operands of the
//                  weights' gradient, are read in place instead of transposed first.  The
//                  32-byte unit u of row r (16 columns) lies in unit u ^ f(r) with f
//                  distinct over the rows that a read touches together: no bank conflicts.
// MXFP4: v_mfma_scale_f32_16x16x128_f8f6f4 takes lane l's 32 codes (row l%16, the 16-byte
// chunk l/16: one block) and that block's scale from a byte of a register, so one
// instruction applies both operands' scales to its exact products and f32 sums.
//
// Accumulator block: register r of lane l holds C row l%16, column 4*(l/16) + r (B's
// fragment is the first operand).
#include "mma_kernel.h"

namespace gk {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
#define GK_LDS(T, p) ((__attribute__((address_space(3))) T *)(p))

// ---------------------------------------------------------------- groups

// Inclusive scans over the wave.
__device__ __forceinline__ int scan_max(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int t = __shfl_up(v, d);
        if (lane >= d) v = v > t ? v : t;
    }
    return v;
}
__device__ __forceinline__ int scan_add(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int t = __shfl_up(v, d);
        if (lane >= d) v += t;
    }
    return v;
}
__device__ __forceinline__ int clamp_row(int v, int M) { return v < 0 ? 0 : (v > M ? M : v); }

// Lane l's group base + l: its rows [s, e), `top` the largest offset before the 64
// groups (then behind them).  Lanes past the last group get an empty range.
__device__ __forceinline__ void group_rows(const int32_t *off, int G, int M, int base, int lane,
                                           int &top, int &s, int &e) {
    const int i = base + lane;
    int lo = i < G ? off[i] : 0, hi = i < G ? off[i + 1] : 0;
    int m = scan_max(lo, lane);
    m = m > top ? m : top;
    s = clamp_row(m, M);
    hi = hi > m ? hi : m;
    e = i < G ? clamp_row(hi, M) : s;
    top = __shfl(hi, 63);
}

struct GroupTile {
    int g;            // group
    int row0, rows;   // the tile's first row and how many rows it has
    int tn;           // tile column
};

// The tile of workgroup `bid`: the groups' tiles in order, a group's in tile_coords order.
// Every workgroup adds up the groups' tile counts itself (G + 1 offsets, in L2 after the
// first), so that nothing has to run before the product.  False: no tile left.
template <int BM>
__device__ __forceinline__ bool find_tile(const int32_t *off, int G, int M, int tiles_n,
                                          int64_t bid, int lane, GroupTile &t) {
    int g = 0, s = 0, e = M, pid, tm_all;
    if (!off) {
        tm_all = (M + BM - 1) / BM;
        const int64_t all = (int64_t)tm_all * tiles_n;
        if (bid >= all) return false;
        pid = (int)xcd_logical(bid, all);
    } else {
        int top = 0, ls = 0, le = 0, incl = 0, total = 0;
        for (int base = 0; base < G; base += 64) {
            group_rows(off, G, M, base, lane, top, ls, le);
            incl = total + scan_add((le - ls + BM - 1) / BM, lane);
            total = __shfl(incl, 63);
        }
        const int64_t all = (int64_t)total * tiles_n;
        if (bid >= all) return false;
        pid = (int)xcd_logical(bid, all);
        if (G > 64) {
            top = total = 0;
            for (int base = 0;; base += 64) {
                group_rows(off, G, M, base, lane, top, ls, le);
                incl = total + scan_add((le - ls + BM - 1) / BM, lane);
                total = __shfl(incl, 63);
                g = base;
                if (pid < total * tiles_n) break;
            }
        }
        // the first lane whose tiles reach past pid (one does: pid is below the total)
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl * tiles_n > pid));
        g += l;
        s = __builtin_amdgcn_readlane(ls, l);
        e = __builtin_amdgcn_readlane(le, l);
        tm_all = (e - s + BM - 1) / BM;
        pid -= (__builtin_amdgcn_readlane(incl, l) - tm_all) * tiles_n;
    }
    int tm, tn;
    tile_coords(pid, tm_all, tiles_n, tm, tn);
    t.g = __builtin_amdgcn_readfirstlane(g);
    t.row0 = __builtin_amdgcn_readfirstlane(s + tm * BM);
    t.rows = __builtin_amdgcn_readfirstlane(e - (s + tm * BM) < BM ? e - (s + tm * BM) : BM);
    t.tn = __builtin_amdgcn_readfirstlane(tn);
    return true;
}

// The rows [s, e) of one group.
__device__ __forceinline__ void one_group(const int32_t *off, int G, int M, int g, int lane,
                                          int &s, int &e) {
    int m = off[0];
    for (int i = lane; i <= g; i += 64) m = off[i] > m ? off[i] : m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int t = __shfl_xor(m, d);
        m = m > t ? m : t;
    }
    const int hi = off[g + 1];
    s = __builtin_amdgcn_readfirstlane(clamp_row(m, M));
    e = __builtin_amdgcn_readfirstlane(clamp_row(hi > m ? hi : m, M));
}

// ---------------------------------------------------------------- stages

// f(r) of a transposed stage of W columns: the eight rows that 32 lanes of a transposing
// read touch (r%4 and bit 3 differ) get units in different banks.  Rows are 2*W bytes:
// below 128 columns several of them share the 64 banks and need fewer different units.
template <int W>
__device__ __forceinline__ int tr_unit(int row) {
    if constexpr (W >= 256) return (row & 3) | (((row >> 3) & 3) << 2);
    if constexpr (W == 128) return (row & 3) | (((row >> 3) & 1) << 2);
    if constexpr (W == 64) return ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
    return (row >> 3) & 1;
}

// A pointer the compiler keeps in scalar registers (a buffer resource built from vector
// registers costs a loop over the lanes for every load).
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const uint8_t *)((uint64_t)hi << 32 | lo);
}

// One operand of a tile: W rows (or columns, TR) of it, filled by NW waves.  Stages are
// loaded in order; `base`, `num` and `left` move on with them.
template <bool TR, int W, int NW>
struct Panel {
    static constexpr int BYTES = W * 128;             // of a stage, either layout
    static constexpr int NI = BYTES / 1024;           // load instructions per stage
    static constexpr int LP = (NI + NW - 1) / NW;     // ... per wave
    const uint8_t *base;  // of the next stage
    int ld;
    uint32_t num;         // k-contiguous: resource size from base
    int left;             // of the contraction from the next stage on: bytes, or rows (TR)
    uint32_t vo[LP];      // this lane's offsets from the stage's base
    int wave, lane;

    // `cols`: bytes of the matrix's columns from the tile's first one (TR).
    __device__ __forceinline__ void init(const uint8_t *b, int64_t ld_, int rows, int k, int cols,
                                         int wave_, int lane_) {
        base = uniform(b);
        ld = (int)ld_;
        wave = wave_;
        lane = lane_;
        left = k;
        num = TR ? 0 : (uint32_t)((rows - 1) * ld + k);
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            const int at = (wave * LP + i) * 64 + lane;  // 16-byte slot of the stage
            if constexpr (TR) {
                const int row = at / (W / 8), slot = at % (W / 8);
                const int ch = ((((slot >> 1) ^ tr_unit<W>(row)) << 1) | (slot & 1)) * 16;
                vo[i] = ch < cols && wave * LP + i < NI ? (uint32_t)(row * ld + ch) : kOutOfRange;
            } else {
                const int row = at / 8;
                vo[i] = wave * LP + i < NI ? (uint32_t)(row * ld + (((at % 8) ^ swz_of<128>(row)) * 16))
                                           : kOutOfRange;
            }
        }
    }
    // Load i of the next stage into the slot at `dst` (waves without one: zeros into
    // `spare`).
    __device__ __forceinline__ void load(uint8_t *dst, uint8_t *spare, int i) const {
        uint8_t *d = NI % NW == 0 || wave * LP + i < NI ? dst + (wave * LP + i) * 1024 : spare;
        if constexpr (TR) {
            // (rows at and past the end read zeros: their offsets reach left * ld)
            dma16(base, size(), vo[i], d);
        } else {
            uint32_t v = vo[i];
            if (left < 128) {  // the K tail's chunks read zeros
                const int slot = (wave * LP + i) * 64 + lane;
                if (((slot % 8) ^ swz_of<128>(slot / 8)) * 16 >= left) v = kOutOfRange;
            }
            dma16(base, size(), v, d);
        }
    }
    // The resource's size for the next stage.
    __device__ __forceinline__ uint32_t size() const {
        return __builtin_amdgcn_readfirstlane(
            TR ? (left >= 64 ? kMaxRecords : (left > 0 ? (uint32_t)(left * ld) : 0))
               : (left > 0 ? num : 0));
    }
    __device__ __forceinline__ void next() {
        if constexpr (TR) {
            base += (int64_t)64 * ld;
            left -= 64;
        } else {
            base += 128;
            num -= 128;
            left -= 128;
        }
    }
};

// Fragments of 16-row (16-column, TR) blocks from a stage.
template <bool TR, int W>
struct Frag {
    int at;
    __device__ __forceinline__ void init(int lane, int first) {
        const int l16 = lane & 15, lq = lane >> 4;
        if constexpr (TR) {
            const int row = 8 * lq + (l16 >> 2);
            at = row * 2 * W + (l16 & 3) * 8 + ((tr_unit<W>(row) ^ (first >> 4)) << 5);
        } else {
            at = (first + l16) * 128 + ((lq ^ swz_of<128>(l16)) << 4);
        }
    }
    // Block j (16*j past `first`, itself a multiple of the blocks a wave reads), half `ss`
    // of the stage.
    __device__ __forceinline__ v4i read(const uint8_t *s, int j, int ss) const {
        if constexpr (TR) {
            const uint8_t *p = s + (at ^ (j << 5)) + 32 * ss * 2 * W;
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(GK_LDS(v4s, p));
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(GK_LDS(v4s, p + 4 * 2 * W));
            const v2i l = __builtin_bit_cast(v2i, lo), h = __builtin_bit_cast(v2i, hi);
            return v4i{l[0], l[1], h[0], h[1]};
        } else {
            return *(const v4i *)(s + (at ^ (ss << 6)) + j * 16 * 128);
        }
    }
};

// Scales of 64 rows (four 16-row blocks) for one stage.  Lane l has read row l's eight
// bytes: x and y, the blocks of the stage's two halves.  The instruction wants, in lane
// 16*q + r, block q's scale of row 16*j + r: a transposition of 4 x 4 bytes among the
// lanes 16 apart, done on both words at once by two swaps of half rows.  Afterwards half
// ss's scale for 16-row block j is byte 2*ss + j/2 of q[j%2].
struct ScaleQuad {
    int q[2];
    __device__ __forceinline__ void set(uint32_t x, uint32_t y) {
        const uint32_t u = __builtin_amdgcn_perm(y, x, 0x05040100);  // x.lo, y.lo
        const uint32_t v = __builtin_amdgcn_perm(y, x, 0x07060302);  // x.hi, y.hi
        const v2u p = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(u, v, false, false));
        const uint32_t a = __builtin_amdgcn_perm(p[1], p[0], 0x06020400);
        const uint32_t b = __builtin_amdgcn_perm(p[1], p[0], 0x07030501);
        const v2u r = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(a, b, false, false));
        q[0] = (int)r[0];
        q[1] = (int)r[1];
    }
};

template <int BA, int BB>
__device__ __forceinline__ v4f mx_step(v4i b, v4i a, v4f c, int sb, int sa) {
    const v8i b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b8, a8, c, 4, 4, BB, sb, BA, sa);
}

__device__ __forceinline__ v4f bf_step(v4i b, v4i a, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b),
                                                   __builtin_bit_cast(v8bf, a), c, 0, 0, 0);
}

// ---------------------------------------------------------------- kernel

// LDS of a tile: the ring, the scale ring (MXFP4: two stages a slot) and 1 KiB that the
// waves without a load of an instruction fill with zeros.
template <bool MX, int BM, int BN, int NS>
struct RaggedLds {
    static constexpr int STAGE = (BM + BN) * 128;
    static constexpr int SA_ROWS = (BM + 63) / 64 * 64, SB_ROWS = (BN + 63) / 64 * 64;
    static constexpr int SSLOT = MX ? (SA_ROWS + SB_ROWS) * 16 : 0;
    static constexpr int NSS = NS / 2 + 1;
    static constexpr int SCALES = NS * STAGE;
    static constexpr int SPARE = SCALES + NSS * SSLOT;
    static constexpr int BYTES = SPARE + 1024;
};

// Waves per SIMD of the workgroups that the LDS holds.
constexpr int ragged_waves(int lds, int nw) {
    const int wgs = 160 * 1024 / lds;
    const int w = wgs * nw / 4;
    return w < 1 ? 1 : (w > 4 ? 4 : w);
}

template <bool MX, bool AT, bool BT, EpiKind E, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(WM * WN * 64)
__attribute__((amdgpu_waves_per_eu(ragged_waves(RaggedLds<MX, BM, BN, NS>::BYTES, WM * WN),
                                   ragged_waves(RaggedLds<MX, BM, BN, NS>::BYTES, WM * WN))))
void ragged_kernel(const RaggedArgs g, const EpiParams ep) {
    static_assert(!MX || (!AT && !BT), "MXFP4 operands are k-contiguous");
    static_assert(!AT || BT, "A transposed: the weights' gradient");
    constexpr int NW = WM * WN;
    constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr int QA = (TM + 3) / 4, QB = (TN + 3) / 4;
    using L = RaggedLds<MX, BM, BN, NS>;
    using PA = Panel<AT, BM, NW>;
    using PB = Panel<BT, BN, NW>;
    constexpr int LPW = PA::LP + PB::LP;  // loads per wave and stage (without scales)
    constexpr int EPI_LD = WTN + 4;
    static_assert(L::BYTES <= 160 * 1024 && NW * 16 * EPI_LD * 4 <= L::BYTES, "LDS");
    static_assert(!MX || (L::SA_ROWS + L::SB_ROWS) / 64 <= NW, "one scale load per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int tiles_n = (g.N + BN - 1) / BN;
    const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;

    GroupTile t;
    int k, z = 0;   // contraction: bytes (k-contiguous A), rows (wgrad)
    const uint8_t *pa = (const uint8_t *)g.a, *pb = (const uint8_t *)g.b;
    if constexpr (AT) {
        const int tiles_m = (g.K + BM - 1) / BM, per = tiles_m * tiles_n;
        const int64_t all = (int64_t)per * g.G;
        if (bid >= all) return;
        const int64_t pid = xcd_logical(bid, all);
        int tm, s, e;
        t.g = (int)(pid / per);
        tile_coords((int)(pid % per), tiles_m, tiles_n, tm, t.tn);
        one_group(g.off, g.G, g.M, t.g, lane, s, e);
        t.row0 = tm * BM;
        t.rows = g.K - t.row0 < BM ? g.K - t.row0 : BM;
        k = e - s;
        z = t.g;
        pa += s * g.lda + (int64_t)t.row0 * 2;
        pb += s * g.ldb;
    } else {
        if (!find_tile<BM>(g.off, g.G, g.M, tiles_n, bid, lane, t)) return;
        k = MX ? (g.K + 31) / 32 * 16 : (g.K * 2 + 15) / 16 * 16;
        pa += t.row0 * g.lda;
        pb += t.g * g.bsb;
    }
    const int n0 = t.tn * BN;
    const int cols = g.N - n0 < BN ? g.N - n0 : BN;
    pb += BT ? (int64_t)n0 * 2 : n0 * g.ldb;
    const int KT = AT ? (k + 63) / 64 : (k + 127) / 128;

    PA A;
    PB B;
    A.init(pa, g.lda, t.rows, k, t.rows * 2, wave, lane);
    // (a transposed B against a k-contiguous A: g.K rows)
    B.init(pb, g.ldb, cols, BT && !AT ? g.K : k, cols * 2, wave, lane);
    uint8_t *const spare = smem + L::SPARE;

    // Scales: wave w loads rows 64*w .. +63 of the tile's A rows and B rows, 16 bytes each
    // (two stages).
    const uint8_t *s_base = nullptr;
    int s_left = 0;  // blocks of a row from the next two stages on
    uint32_t s_vo = 0;
    const int nb = (g.K + 31) / 32;  // blocks of a row
    if constexpr (MX) {
        constexpr int NA = L::SA_ROWS / 64;
        const bool is_a = wave < NA;
        const int r0 = (is_a ? wave : wave - NA) * 64;
        const int64_t lds = is_a ? g.lsa : g.lsb;
        s_base = uniform(is_a ? g.sa + (t.row0 + r0) * lds
                              : g.sb + t.g * g.bssb + (int64_t)(n0 + r0) * lds);
        const int rows = wave >= (L::SA_ROWS + L::SB_ROWS) / 64 ? 0 : (is_a ? t.rows : cols) - r0;
        s_left = rows > 0 ? nb : 0;
        s_vo = lane < rows ? (uint32_t)(lane * (int)lds) : kOutOfRange;
    }
    int s_slot = 0;
    auto load_scales = [&]() {  // of the next two stages
        uint8_t *d = wave < (L::SA_ROWS + L::SB_ROWS) / 64
                         ? smem + L::SCALES + s_slot * L::SSLOT + wave * 1024
                         : spare;
        dma16(s_base, __builtin_amdgcn_readfirstlane(s_left > 0 ? kMaxRecords : 0), s_vo, d);
        s_base += 16;
        s_left -= 16;
        s_slot = s_slot == L::NSS - 1 ? 0 : s_slot + 1;
    };
    auto load_stage = [&](uint8_t *d) {
#pragma unroll
        for (int i = 0; i < PA::LP; ++i) A.load(d, spare, i);
#pragma unroll
        for (int i = 0; i < PB::LP; ++i) B.load(d + PA::BYTES, spare, i);
        A.next();
        B.next();
    };

    Frag<AT, BM> fa;
    Frag<BT, BN> fb;
    fa.init(lane, wm * WTM);
    fb.init(lane, wn * WTN);
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{};

    int r_slot = 0;  // the scale slot in use
    // Stage kt, in slot kt % NS; PAR: kt's parity.
    auto kstep = [&](int kt, auto par, uint8_t *__restrict__ wr, const uint8_t *__restrict__ sa) {
        constexpr int PAR = decltype(par)::value;
        // Loads in flight behind stage kt's: stages kt+1 .. kt+NS-2, the even ones with
        // their scales.
        constexpr int SC = MX ? (NS - 2 + PAR) / 2 : 0;
        wait_vmcnt<(NS - 2) * LPW + SC>();
        stage_barrier();
        if constexpr (MX && (PAR + NS - 1) % 2 == 0) load_scales();
        load_stage(wr);
        const uint8_t *const sb = sa + PA::BYTES;
        ScaleQuad xa[QA], xb[QB];
        if constexpr (MX) {
            const uint8_t *sc = smem + L::SCALES + r_slot * L::SSLOT + PAR * 8;
            if (PAR) r_slot = r_slot == L::NSS - 1 ? 0 : r_slot + 1;
            // A row's bytes past its blocks hold anything: cleared, so that no NaN
            // scale meets the zero codes there.
            const int nv = nb - kt * 8;
            const uint32_t mx = nv >= 4 ? ~0u : (1u << (8 * nv)) - 1;
            const uint32_t my = nv >= 8 ? ~0u : (nv <= 4 ? 0u : (1u << (8 * (nv - 4))) - 1);
#pragma unroll
            for (int i = 0; i < QA; ++i) {
                const v2u w = *(const v2u *)(sc + (wm * WTM + 64 * i + (lane & (WTM - 1 < 63 ? WTM - 1 : 63))) * 16);
                xa[i].set(w[0] & mx, w[1] & my);
            }
#pragma unroll
            for (int i = 0; i < QB; ++i) {
                const v2u w = *(const v2u *)(sc + (L::SA_ROWS + wn * WTN + 64 * i + (lane & (WTN - 1 < 63 ? WTN - 1 : 63))) * 16);
                xb[i].set(w[0] & mx, w[1] & my);
            }
        }
        auto half = [&](auto hh) {
            constexpr int SS = decltype(hh)::value;
            v4i af[TM], bf[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) bf[j] = fb.read(sb, j, SS);
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = fa.read(sa, i, SS);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    if constexpr (MX) {
                        // (the byte of a scale register is an immediate)
                        const int x = xa[i / 4].q[i % 2], y = xb[j / 4].q[j % 2];
                        const bool ia = (i / 2) % 2, jb = (j / 2) % 2;
                        acc[i][j] = ia ? (jb ? mx_step<2 * SS + 1, 2 * SS + 1>(bf[j], af[i], acc[i][j], y, x)
                                             : mx_step<2 * SS + 1, 2 * SS>(bf[j], af[i], acc[i][j], y, x))
                                       : (jb ? mx_step<2 * SS, 2 * SS + 1>(bf[j], af[i], acc[i][j], y, x)
                                             : mx_step<2 * SS, 2 * SS>(bf[j], af[i], acc[i][j], y, x));
                    } else {
                        acc[i][j] = bf_step(bf[j], af[i], acc[i][j]);
                    }
                }
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
    };

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        if constexpr (MX) {
            if (s % 2 == 0) load_scales();
        }
        load_stage(smem + s * L::STAGE);
    }
    int slot = 0;
    auto step = [&](int kt, auto par) {
        const int w = slot == 0 ? NS - 1 : slot - 1;
        kstep(kt, par, smem + w * L::STAGE, smem + slot * L::STAGE);
        slot = slot == NS - 1 ? 0 : slot + 1;
    };
    for (int kt = 0; kt < KT; kt += 2) {
        step(kt, std::integral_constant<int, 0>{});
        if (kt + 1 < KT) step(kt + 1, std::integral_constant<int, 1>{});
    }

    // Epilogue: 16-row bands of the wave staged through LDS and stored as rows.  The loads
    // past the end of K (zeros into ring slots) land first.
    wait_vmcnt<0>();
    __syncthreads();
    float *const stg = (float *)smem + wave * 16 * EPI_LD;
    constexpr int CPRE = WTN / 4;                       // 4-element chunks per row
    constexpr int RPIT = 64 / CPRE < 16 ? 64 / CPRE : 16;  // rows per pass
    const int l16 = lane & 15, lq = lane >> 4;
    const int gcol0 = n0 + wn * WTN;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) *(v4f *)(stg + l16 * EPI_LD + j * 16 + 4 * lq) = acc[i][j];
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int it = 0; it < 16 / RPIT; ++it) {
            const int r = it * RPIT + lane / CPRE, c4 = (lane % CPRE) * 4;
            const v4f v4 = *(const v4f *)(stg + r * EPI_LD + c4);
            const float v[4] = {v4[0], v4[1], v4[2], v4[3]};
            const int row = wm * WTM + i * 16 + r;
            if (row < t.rows && gcol0 + c4 < g.N)
                store4<E, float, StPol::Plain>(ep, z, t.row0 + row, gcol0 + c4, g.N, v);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_wave_barrier();
    }
}

// Workgroups go out in rows of at most 2^20 (a grid's x extent counts threads in 32 bits).
inline dim3 ragged_grid(int64_t tiles) {
    constexpr int64_t X = 1 << 20;
    return tiles <= X ? dim3((uint32_t)tiles) : dim3((uint32_t)X, (uint32_t)((tiles + X - 1) / X));
}

// Tiles of a forward product at most: every group's last one may be part of a tile.
inline int64_t ragged_tiles(const RaggedArgs &g, int bm, int bn) {
    const int64_t groups = g.G < g.M ? g.G : g.M;
    const int64_t tm = g.off ? (g.M + groups * (bm - 1)) / bm : (g.M + bm - 1) / bm;
    return tm * ((g.N + bn - 1) / bn);
}

template <bool MX, bool AT, bool BT, EpiKind E, int BM, int BN, int WM, int WN, int NS>
static hipError_t ragged_go(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    // 32-bit offsets inside a panel, with the loads of rows past its edge
    const int64_t kbytes = MX ? (int64_t)(g.K + 31) / 32 * 16 : (int64_t)g.K * 2;
    if ((AT ? 64 : BM) * g.lda + kbytes > (int64_t)kMaxRecords ||
        (BT ? 64 * g.ldb + (int64_t)g.N * 2 : BN * g.ldb + kbytes) > (int64_t)kMaxRecords ||
        (MX && 64 * (g.lsa > g.lsb ? g.lsa : g.lsb) > (int64_t)kMaxRecords))
        return hipErrorInvalidValue;
    const int64_t tiles = AT ? (int64_t)g.G * ((g.K + BM - 1) / BM) * ((g.N + BN - 1) / BN)
                             : ragged_tiles(g, BM, BN);
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((ragged_kernel<MX, AT, BT, E, BM, BN, WM, WN, NS>), ragged_grid(tiles),
                       dim3(WM * WN * 64), 0, stream, g, ep);
    return hipGetLastError();
}

}  // namespace gk
