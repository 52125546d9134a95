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
#include <algorithm>
#include <cmath>

#include "mma_kernel.h"

namespace gk {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
#define GK_LDS(T, p) ((__attribute__((address_space(3))) T *)(p))

// ---------------------------------------------------------------- groups

// Inclusive scans over the wave of non-negative values (0 is neutral for both), in
// registers: shifts within rows of 16 lanes, then each row's last value to the rows after.
template <typename F>
__device__ __forceinline__ int scan(int v, F op) {
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));   // row_shr:1
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));  // row_bcast:15
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));  // row_bcast:31
    return v;
}
__device__ __forceinline__ int scan_max(int v) {
    return scan(v, [](int a, int b) { return a > b ? a : b; });
}
__device__ __forceinline__ int scan_add(int v) {
    return scan(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int clamp_row(int v, int M) { return v < 0 ? 0 : (v > M ? M : v); }

// Lane l's group base + l: its rows [s, e), `top` the largest offset before the 64
// groups (then behind them).  Lanes past the last group get an empty range.
__device__ __forceinline__ void group_rows(const int32_t *off, int G, int M, int base, int lane,
                                           int &top, int &s, int &e) {
    const int i = base + lane;
    int lo = i < G ? off[i] : 0, hi = i < G ? off[i + 1] : 0;
    int m = scan_max(lo > 0 ? lo : 0);
    m = m > top ? m : top;
    s = clamp_row(m, M);
    hi = hi > m ? hi : m;
    e = i < G ? clamp_row(hi, M) : s;
    top = __builtin_amdgcn_readlane(hi, 63);
}

struct GroupTile {
    int g;            // group
    int row0, rows;   // the tile's first row and how many rows it has
    int tn;           // tile column
};

// The tile of workgroup `bid`: the groups' tiles in order, a group's in tile_coords order,
// every XCD a contiguous range of them (xcd_logical).  Every workgroup adds up the groups'
// tile counts itself (G + 1 offsets, in L2 after the first), so that nothing has to run
// before the product.  False: no tile left.
// HALVES: where the tiles of an XCD's last round would leave half of its CUs (cus / 8) or
// more without one, each goes out as two tiles of half the rows.
template <int BM, bool HALVES>
__device__ __forceinline__ bool find_tile(const int32_t *off, int G, int M, int tiles_n, int cus,
                                          int64_t bid, int lane, GroupTile &t) {
    int g = 0, s = 0, e = M, ls = 0, le = 0, incl = 0, total = 0;
    if (!off) {
        total = (M + BM - 1) / BM;
    } else {
        int top = 0;
        for (int base = 0; base < G; base += 64) {
            group_rows(off, G, M, base, lane, top, ls, le);
            incl = total + scan_add((le - ls + BM - 1) / BM);
            total = __builtin_amdgcn_readlane(incl, 63);
        }
    }
    const int all = total * tiles_n;  // (below 2^31: the host checks the upper bound)
    const int xcd = (int)(bid % 8), per = all / 8, rem = all % 8;
    const int mine = per + (xcd < rem ? 1 : 0);
    int idx = (int)(bid / 8), half = -1;
    if constexpr (HALVES) {
        const int cx = cus / 8 > 0 ? cus / 8 : 1, whole = mine / cx * cx;
        if (2 * (mine - whole) <= cx && idx >= whole) {
            half = (idx - whole) & 1;
            idx = whole + (idx - whole) / 2;
        }
    }
    if (idx >= mine) return false;
    int pid = xcd * per + (xcd < rem ? xcd : rem) + idx;
    if (off) {
        if (G > 64) {
            int top = 0;
            total = 0;
            for (int base = 0;; base += 64) {
                group_rows(off, G, M, base, lane, top, ls, le);
                incl = total + scan_add((le - ls + BM - 1) / BM);
                total = __builtin_amdgcn_readlane(incl, 63);
                g = base;
                if (pid < total * tiles_n) break;
                // (Something wrote the offsets while the product runs, and this second
                // reading has fewer tiles than the first.)
                if (G - base <= 64) return false;
            }
        }
        // the first lane whose tiles reach past pid (one does: pid is below the total)
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl * tiles_n > pid));
        g += l;
        s = __builtin_amdgcn_readlane(ls, l);
        e = __builtin_amdgcn_readlane(le, l);
        total = (e - s + BM - 1) / BM;
        pid -= (__builtin_amdgcn_readlane(incl, l) - total) * tiles_n;
    }
    int tm, tn;
    tile_coords(pid, total, tiles_n, tm, tn);
    int row0 = s + tm * BM, rows = e - row0 < BM ? e - row0 : BM;
    if (half >= 0) {
        row0 += half * (BM / 2);
        rows -= half * (BM / 2);
        if (rows <= 0) return false;
        rows = rows < BM / 2 ? rows : BM / 2;
    }
    t.g = __builtin_amdgcn_readfirstlane(g);
    t.row0 = __builtin_amdgcn_readfirstlane(row0);
    t.rows = __builtin_amdgcn_readfirstlane(rows);
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

// dma16 (mma_kernel.h); ONCE: nontemporally, the caches keep nothing of it.
template <bool ONCE>
__device__ __forceinline__ void load16(const uint8_t *base, uint32_t num, uint32_t voff,
                                       uint8_t *lds) {
    constexpr int kNt = 2;  // the instruction's nt bit
    __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, (int)num, kRsrcWord3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                             voff, 0, 0, ONCE ? kNt : 0);
}

// One operand of a tile: W rows (or columns, TR) of it, filled by NW waves.  Stages are
// loaded in order; `base`, `num` and `left` move on with them.
template <bool TR, int W, int NW, bool ONCE = false>
struct Panel {
    static constexpr int BYTES = W * 128;             // of a stage, either layout
    static constexpr int NI = BYTES / 1024;           // load instructions per stage
    static constexpr int LP = (NI + NW - 1) / NW;     // ... per wave
    const uint8_t *base;  // of the next stage
    int ld;
    uint32_t num;         // k-contiguous: resource size from base
    int left;             // of the contraction from the next stage on: bytes, or rows (TR)
    // This lane's offsets from the stage's base: of loads 0 and 1; the layouts repeat
    // after two loads, 2*RPI rows further on.
    static constexpr int RPI = TR ? 1024 / (2 * W) : 8;  // rows one load fills
    static constexpr bool PAIR = TR ? RPI == 2 && LP == 4 : LP % 2 == 0;
    static constexpr int NVO = PAIR ? 2 : LP;
    uint32_t vo[NVO];
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
        for (int i = 0; i < NVO; ++i) {
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
        // (an out-of-range offset stays one with the rows added)
        uint32_t v = PAIR ? vo[i % 2] + (uint32_t)(i / 2 * 2 * RPI * ld) : vo[i];
        if constexpr (TR) {
            // (rows at and past the end read zeros: their offsets reach left * ld)
            load16<ONCE>(base, size(), v, d);
        } else {
            if (left < 128) {  // the K tail's chunks read zeros
                const int slot = (wave * LP + i) * 64 + lane;
                if (((slot % 8) ^ swz_of<128>(slot / 8)) * 16 >= left) v = kOutOfRange;
            }
            load16<ONCE>(base, size(), v, d);
        }
    }
    // The resource's size for the next stage.
    __device__ __forceinline__ uint32_t size() const {
        return __builtin_amdgcn_readfirstlane(
            TR ? (left >= 64 ? kMaxRecords : (left > 0 ? (uint32_t)(left * ld) : 0))
               : (left > 0 ? num : 0));
    }
    __device__ __forceinline__ void skip(int stages) {
        if constexpr (TR) {
            base += (int64_t)stages * 64 * ld;
            left -= stages * 64;
        } else {
            base += stages * 128;
            num -= (uint32_t)stages * 128;
            left -= stages * 128;
        }
    }
    __device__ __forceinline__ void next() { skip(1); }
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
    static constexpr int SSLOT = MX ? ((BM + 63) / 64 + (BN + 63) / 64) * 1024 : 0;
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

// ---------------------------------------------------------------- tiles

// What a workgroup computes.
struct RaggedTile {
    int row0, rows;   // rows of C (wgrad: of C_g) and how many of them
    int n0, cols;     // columns
    int g, z;         // group; batch element of C
    int k;            // contraction: bytes of A (k-contiguous), rows (wgrad)
    int KT;           // stages
    const uint8_t *a, *b;
};

// wgrad: how many workgroups an XCD gets for each group's `per` tiles.
__device__ __host__ __forceinline__ int wgrad_share(int per) { return (per + 7) / 8; }

template <bool MX, bool AT, bool BT, int BM, int BN, bool HALVES>
__device__ __forceinline__ bool ragged_tile(const RaggedArgs &g, int lane, RaggedTile &t) {
    const int tiles_n = (g.N + BN - 1) / BN;
    const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    t.a = (const uint8_t *)g.a;
    t.b = (const uint8_t *)g.b;
    t.z = 0;
    int tn;
    if constexpr (AT) {
        // Every XCD takes an eighth of each group's tiles, a contiguous one: with whole
        // groups per XCD the one with the longest group would work on alone.  (The
        // eighths turn with the group, so that their roundings even out.)
        const int tiles_m = (g.K + BM - 1) / BM, tiles = tiles_m * tiles_n;
        const int per = tiles * g.splits, share = wgrad_share(per);
        const int64_t idx = bid / 8;
        t.g = (int)(idx / share);
        if (t.g >= g.G) return false;
        const int part = (int)((bid + t.g) % 8);
        const int pid = (int)((int64_t)part * per / 8) + (int)(idx % share);
        if (pid >= (int)((int64_t)(part + 1) * per / 8)) return false;
        int tm, s, e;
        tile_coords(pid % tiles, tiles_m, tiles_n, tm, tn);
        s = 0;
        e = g.M;
        if (g.off) one_group(g.off, g.G, g.M, t.g, lane, s, e);
        const int sp = pid / tiles;
        if (g.splits > 1) {  // this part's stages of the group
            const int stages = (e - s + 63) / 64;
            const int lo = (int)((int64_t)stages * sp / g.splits);
            const int hi = (int)((int64_t)stages * (sp + 1) / g.splits);
            e = e < s + hi * 64 ? e : s + hi * 64;
            s += lo * 64;
        }
        t.row0 = tm * BM;
        t.rows = g.K - t.row0 < BM ? g.K - t.row0 : BM;
        t.k = e > s ? e - s : 0;
        t.z = t.g * g.splits + sp;
        t.KT = (t.k + 63) / 64;
        t.a += s * g.lda + (int64_t)t.row0 * 2;
        t.b += s * g.ldb;
    } else {
        GroupTile f;
        if (!find_tile<BM, HALVES>(g.off, g.G, g.M, tiles_n, g.cus, bid, lane, f)) return false;
        t.g = f.g;
        t.row0 = f.row0;
        t.rows = f.rows;
        tn = f.tn;
        t.k = MX ? (g.K + 31) / 32 * 16 : (g.K * 2 + 15) / 16 * 16;
        t.KT = (t.k + 127) / 128;
        t.a += t.row0 * g.lda;
        t.b += t.g * g.bsb;
    }
    t.n0 = tn * BN;
    t.cols = g.N - t.n0 < BN ? g.N - t.n0 : BN;
    t.b += BT ? (int64_t)t.n0 * 2 : t.n0 * g.ldb;
    return true;
}

// The scales of a MXFP4 tile: wave w loads rows 64*w .. +63 of the tile's A rows, then of
// its B rows, 16 bytes each (two stages) at a time.
template <int BM, int BN>
struct ScalePanel {
    static constexpr int A_ROWS = (BM + 63) / 64 * 64, B_ROWS = (BN + 63) / 64 * 64;
    static constexpr int SLOT = (A_ROWS + B_ROWS) * 16;
    const uint8_t *base;
    int left;       // blocks of a row from the next two stages on
    uint32_t vo;
    uint8_t *dst;   // this wave's part of slot 0
    bool mine;

    __device__ __forceinline__ void init(const RaggedArgs &g, const RaggedTile &t, uint8_t *slots,
                                         uint8_t *spare, int wave, int lane) {
        constexpr int NA = A_ROWS / 64;
        const bool is_a = wave < NA;
        const int r0 = (is_a ? wave : wave - NA) * 64;
        const int64_t lds = is_a ? g.lsa : g.lsb;
        base = uniform(is_a ? g.sa + (t.row0 + r0) * lds
                            : g.sb + t.g * g.bssb + (int64_t)(t.n0 + r0) * lds);
        mine = wave < (A_ROWS + B_ROWS) / 64;
        const int rows = mine ? (is_a ? t.rows : t.cols) - r0 : 0;
        left = rows > 0 ? (g.K + 31) / 32 : 0;
        vo = lane < rows ? (uint32_t)(lane * (int)lds) : kOutOfRange;
        dst = mine ? slots + wave * 1024 : spare;
    }
    __device__ __forceinline__ void load(int slot) {
        dma16(base, __builtin_amdgcn_readfirstlane(left > 0 ? kMaxRecords : 0), vo,
              mine ? dst + slot * SLOT : dst);
        base += 16;
        left -= 16;
    }
};

// The scales of N 64-row quads of a wave for one stage: rows from `row` of the slot at sc
// (+ 8 in an odd stage); `nv` blocks of the row remain from this stage on.
template <int N, int ROWS>
__device__ __forceinline__ void read_scales(const uint8_t *sc, int row, int nv, int lane,
                                            ScaleQuad (&x)[N]) {
    // A row's bytes past its blocks hold anything: cleared, so that no NaN scale meets the
    // zero codes there.
    const uint32_t mx = nv >= 4 ? ~0u : (nv <= 0 ? 0u : (1u << (8 * nv)) - 1);
    const uint32_t my = nv >= 8 ? ~0u : (nv <= 4 ? 0u : (1u << (8 * (nv - 4))) - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const v2u w = *(const v2u *)(sc + (row + 64 * i + (lane & (ROWS < 64 ? ROWS - 1 : 63))) * 16);
        x[i].set(w[0] & mx, w[1] & my);
    }
}

// A row's last block may hold codes past its k columns, which do not count: cleared in the W
// rows of one operand of that stage, in LDS (a code of zero makes the other operand's
// products there zero whatever they are).  Thread r does row r.  The kernels run that stage
// behind their loops: a test in every stage costs up to 5% (and the 256 x 256 tile spills).
template <int W>
__device__ __forceinline__ void mx_cut(uint8_t *stage, int r, int k) {
    if (r >= W) return;
    v4i *const p = (v4i *)(stage + r * 128 + (((k >> 5 & 7) ^ swz_of<128>(r)) << 4));
    v4i v = *p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = (k & 31) - 8 * i;  // codes of this word that count
        v[i] = n >= 8 ? v[i] : (n <= 0 ? 0 : v[i] & ((1 << (4 * n)) - 1));
    }
    *p = v;
}

// acc[i][j] += the products of half SS of a stage.
template <int SS>
__device__ __forceinline__ v4f mx_half(v4i b, v4i a, v4f c, const ScaleQuad &y, const ScaleQuad &x,
                                       int i, int j) {
    // (the byte of a scale register is an immediate)
    const int sx = x.q[i % 2], sy = y.q[j % 2];
    const bool ia = (i / 2) % 2, jb = (j / 2) % 2;
    return ia ? (jb ? mx_step<2 * SS + 1, 2 * SS + 1>(b, a, c, sy, sx)
                    : mx_step<2 * SS + 1, 2 * SS>(b, a, c, sy, sx))
              : (jb ? mx_step<2 * SS, 2 * SS + 1>(b, a, c, sy, sx)
                    : mx_step<2 * SS, 2 * SS>(b, a, c, sy, sx));
}

// Elements a lane stores at once: 16 bytes.
constexpr int chunk_of(EpiKind e) { return e == EpiKind::BF16 ? 8 : 4; }

// Whether C's rows start at 128-byte lines.
template <EpiKind E>
__device__ __forceinline__ bool whole_lines(const EpiParams &ep) {
    constexpr int ESZ = E == EpiKind::BF16 ? 2 : 4;
    return (((uint64_t)ep.c | (uint64_t)(ep.rsc * ESZ) | (uint64_t)(ep.bsc * ESZ)) & 127) == 0;
}

// A chunk of one row of C; NT: stored nontemporally.  Written through the L2 the output
// pushes the operand panels out of it (weight gradients in turn on one card: 16384x8x4096x4096
// with f32 output 519 against 459 us, 1003x32x1024x704 with bf16 output 18.8 against 16.0), but
// pieces of lines have to meet there (rows of 9632 bytes, 39x56x512x2408: 97 us
// nontemporally, 60 without).  bf16 takes 16 bytes here instead of
// store4's 8: a weight gradient of short groups is bound by its stores (32 x 1024 x 1024 bf16
// from 64 rows: 21.8 us with 8 bytes a lane).
template <EpiKind E, bool NT>
__device__ __forceinline__ void store_chunk(const EpiParams &ep, int64_t z, int row, int col, int N,
                                            const v4f (&v)[chunk_of(E) / 4]) {
    if constexpr (E == EpiKind::BF16) {
        if (ep.vec4 && col + 8 <= N) {
            typedef uint32_t v4u __attribute__((ext_vector_type(4)));
            typedef uint32_t v4u_any2 __attribute__((ext_vector_type(4), aligned(2)));
            uint16_t *c = (uint16_t *)ep.c + z * ep.bsc + (int64_t)row * ep.rsc + col;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = ep.alpha_f * v[e / 4][e % 4];
            if (ep.beta_f != 0.0f) {
                const v4u old = *(const v4u_any2 *)c;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = bf16_widen((uint16_t)(old[e / 2] >> (16 * (e % 2))));
                    f[e] = ep.beta_f == 1.0f ? w + f[e] : __builtin_fmaf(ep.beta_f, w, f[e]);
                }
            }
            v4u o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = bf16x2_rne(f[2 * e], f[2 * e + 1]);
            if constexpr (NT) __builtin_nontemporal_store(o, (v4u_any2 *)c);
            else *(v4u_any2 *)c = o;
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < chunk_of(E) / 4; ++i) {
        const float w[4] = {v[i][0], v[i][1], v[i][2], v[i][3]};
        if (col + 4 * i < N)
            store4<E, float, NT ? StPol::NT : StPol::Plain>(ep, z, row, col + 4 * i, N, w);
    }
}

// Epilogue: 16-row bands of a wave's TM x TN blocks staged through LDS and stored as rows.
template <EpiKind E, bool NT, int WTM, int WTN, int TM, int TN>
__device__ __forceinline__ void ragged_store(const EpiParams &ep, const RaggedTile &t, int N,
                                             const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                             int wm, int wn, int lane) {
    constexpr int LD = WTN + 4, CH = chunk_of(E);
    constexpr int CPR = WTN / CH;                        // chunks per row
    constexpr int RPP = 64 / CPR < 16 ? 64 / CPR : 16;   // rows per pass
    float *const stg = (float *)smem + wave * 16 * LD;
    const int l16 = lane & 15, lq = lane >> 4;
    const int r0 = lane / CPR, c = lane % CPR * CH, col = t.n0 + wn * WTN + c;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) *(v4f *)(stg + l16 * LD + j * 16 + 4 * lq) = acc[i][j];
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int r = r0; r < 16; r += RPP) {
            v4f v[CH / 4];
#pragma unroll
            for (int e = 0; e < CH / 4; ++e) v[e] = *(const v4f *)(stg + r * LD + c + 4 * e);
            const int row = wm * WTM + i * 16 + r;
            if (row < t.rows && col < N) store_chunk<E, NT>(ep, t.z, t.row0 + row, col, N, v);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_wave_barrier();
    }
}

// The sums of the KS waves that share a BM x BN tile, added in wave order and stored.
template <EpiKind E, bool NT, int BM, int BN, int KS, int TM, int TN>
__device__ __forceinline__ void wave_sums(const EpiParams &ep, const RaggedTile &t, int N,
                                          const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                          int lane) {
    constexpr int LD = BN + 4, CH = chunk_of(E);
    float *const sums = (float *)smem;
    const int l16 = lane & 15, lq = lane >> 4;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            *(v4f *)(sums + (wave * BM + i * 16 + l16) * LD + j * 16 + 4 * lq) = acc[i][j];
    __syncthreads();
#pragma unroll 1
    for (int c = threadIdx.x; c < BM * BN / CH; c += KS * 64) {
        const int row = c / (BN / CH), col = c % (BN / CH) * CH;
        if (row >= t.rows || t.n0 + col >= N) continue;
        v4f v[CH / 4] = {};
#pragma unroll
        for (int w = 0; w < KS; ++w)
#pragma unroll
            for (int i = 0; i < CH / 4; ++i)
                v[i] += *(const v4f *)(sums + (w * BM + row) * LD + col + 4 * i);
        store_chunk<E, NT>(ep, t.z, t.row0 + row, t.n0 + col, N, v);
    }
}

// How a tile leaves the kernels: tile() of waves that each hold WTM x WTN of it, waves() of
// waves that each hold sums of all of it, with SMEM bytes of LDS that nothing else uses any
// more.  EarlyTile and EarlyWaves hold what these read from memory beside the products,
// loaded behind the first stages' loads.  PlainOut: EpiParams' map.
template <EpiKind E>
struct PlainOut {
    using Params = EpiParams;
    struct Nothing {
        __device__ __forceinline__ void load(const Params &, const RaggedTile &, int, int, int) {}
    };
    template <int BM, int BN, int WM, int WN>
    using EarlyTile = Nothing;
    template <int BM, int BN, int KS>
    using EarlyWaves = Nothing;
    template <int BM, int BN, int WM, int WN, int SMEM, int TM, int TN>
    __device__ __forceinline__ static void tile(const Params &ep, const RaggedTile &t, int N,
                                                const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                                int lane, const Nothing &) {
        constexpr int WTM = BM / WM, WTN = BN / WN;
        const int wm = wave / WN, wn = wave % WN;
        if (whole_lines<E>(ep)) ragged_store<E, true, WTM, WTN>(ep, t, N, acc, smem, wave, wm, wn, lane);
        else ragged_store<E, false, WTM, WTN>(ep, t, N, acc, smem, wave, wm, wn, lane);
    }
    template <int BM, int BN, int KS, int SMEM, int TM, int TN>
    __device__ __forceinline__ static void waves(const Params &ep, const RaggedTile &t, int N,
                                                 const v4f (&acc)[TM][TN], uint8_t *smem, int wave,
                                                 int lane, const Nothing &) {
        if (whole_lines<E>(ep)) wave_sums<E, true, BM, BN, KS>(ep, t, N, acc, smem, wave, lane);
        else wave_sums<E, false, BM, BN, KS>(ep, t, N, acc, smem, wave, lane);
    }
};

// ---------------------------------------------------------------- small tiles

// BM x BN tiles on a ring of NS stages: stage kt + NS - 1 is loaded while kt is multiplied, one
// barrier a stage.  Bound by loads in flight where groups are short: 16 x 64, nontemporal, reads
// 64x32x2048x4096's 4-bit weights (107 MB of the 24 groups that have rows) in 21.9 us, 4.9 TB/s;
// small outputs leave the CUs' matrix cores waiting for their first stages (1003x32x1024x704's
// weight gradient 16.0 us, 2.9 TB/s of stores).
template <bool MX, bool AT, bool BT, typename O, int BM, int BN, int WM, int WN, int NS, bool ONCE>
__global__ __launch_bounds__(WM * WN * 64)
__attribute__((amdgpu_waves_per_eu(ragged_waves(RaggedLds<MX, BM, BN, NS>::BYTES, WM * WN),
                                   ragged_waves(RaggedLds<MX, BM, BN, NS>::BYTES, WM * WN))))
void ragged_kernel(const RaggedArgs g, const typename O::Params ep) {
    static_assert(!MX || (!AT && !BT), "MXFP4 operands are k-contiguous");
    static_assert(!AT || BT, "A transposed: the weights' gradient");
    constexpr int NW = WM * WN;
    constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr int QA = (TM + 3) / 4, QB = (TN + 3) / 4;
    using L = RaggedLds<MX, BM, BN, NS>;
    using PA = Panel<AT, BM, NW>;
    using PB = Panel<BT, BN, NW, ONCE>;
    using SP = ScalePanel<BM, BN>;
    constexpr int LPW = PA::LP + PB::LP;  // loads per wave and stage (without scales)
    static_assert(L::BYTES <= 160 * 1024 && NW * 16 * (WTN + 4) * 4 <= L::BYTES, "LDS");
    static_assert(!MX || (SP::A_ROWS + SP::B_ROWS) / 64 <= NW, "one scale load per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    RaggedTile t;
    if (!ragged_tile<MX, AT, BT, BM, BN, false>(g, lane, t)) return;

    PA A;
    PB B;
    A.init(t.a, g.lda, t.rows, t.k, t.rows * 2, wave, lane);
    // (a transposed B against a k-contiguous A: g.K rows)
    B.init(t.b, g.ldb, t.cols, BT && !AT ? g.K : t.k, t.cols * 2, wave, lane);
    uint8_t *const spare = smem + L::SPARE;
    SP S;
    if constexpr (MX) S.init(g, t, smem + L::SCALES, spare, wave, lane);
    const int nb = (g.K + 31) / 32;  // blocks of a row
    int s_slot = 0, r_slot = 0;      // scale slots: the next to fill, the one in use
    auto load_scales = [&]() {  // of the next two stages
        S.load(s_slot);
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

    ScaleQuad xa[QA], xb[QB];
    auto scales = [&](int kt, int par) {  // of stage kt, which has landed
        const uint8_t *sc = smem + L::SCALES + r_slot * SP::SLOT + par * 8;
        read_scales<QA, WTM>(sc, wm * WTM, nb - kt * 8, lane, xa);
        read_scales<QB, WTN>(sc, SP::A_ROWS + wn * WTN, nb - kt * 8, lane, xb);
    };
    auto half = [&](const uint8_t *sa, const uint8_t *sb, auto hh) {
        constexpr int SS = decltype(hh)::value;
        v4i af[TM], bf[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) bf[j] = fb.read(sb, j, SS);
#pragma unroll
        for (int i = 0; i < TM; ++i) af[i] = fa.read(sa, i, SS);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = MX ? mx_half<SS>(bf[j], af[i], acc[i][j], xb[j / 4], xa[i / 4], i, j)
                               : bf_step(bf[j], af[i], acc[i][j]);
    };
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;
    // Stage kt; PAR: kt's parity.  wr: the slot to load into, sa: the stage's own.  The two
    // differ, and `restrict` says so: else the compiler waits for every load in flight
    // before the transposing reads.
    auto kstep = [&](int kt, auto par, uint8_t *__restrict__ wr, const uint8_t *__restrict__ sa) {
        constexpr int PAR = decltype(par)::value;
        // Loads in flight behind stage kt's: stages kt+1 .. kt+NS-2, the even ones with
        // their scales.
        constexpr int SC = MX ? (NS - 2 + PAR) / 2 : 0;
        wait_vmcnt<(NS - 2) * LPW + SC>();
        stage_barrier();
        if constexpr (MX && (PAR + NS - 1) % 2 == 0) load_scales();
        load_stage(wr);
        if constexpr (MX) {
            scales(kt, PAR);
            if (PAR) r_slot = r_slot == L::NSS - 1 ? 0 : r_slot + 1;
        }
        half(sa, sa + PA::BYTES, H0{});
        half(sa, sa + PA::BYTES, H1{});
    };

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        if constexpr (MX) {
            if (s % 2 == 0) load_scales();
        }
        load_stage(smem + s * L::STAGE);
    }
    typename O::template EarlyTile<BM, BN, WM, WN> early;
    early.load(ep, t, g.N, wave, lane);
    int slot = 0;
    auto step = [&](int kt, auto par) {
        const int w = slot == 0 ? NS - 1 : slot - 1;
        kstep(kt, par, smem + w * L::STAGE, smem + slot * L::STAGE);
        slot = slot == NS - 1 ? 0 : slot + 1;
    };
    const int whole = MX && g.K % 32 ? t.KT - 1 : t.KT;  // stages without a cut block
    for (int kt = 0; kt < whole; kt += 2) {
        step(kt, H0{});
        if (kt + 1 < whole) step(kt + 1, H1{});
    }

    // (the loads past the end of K, zeros into ring slots, land first)
    wait_vmcnt<0>();
    __syncthreads();
    if (MX && whole < t.KT) {
        uint8_t *const sa = smem + slot * L::STAGE;
        mx_cut<BM>(sa, threadIdx.x, g.K);
        __syncthreads();
        scales(whole, whole & 1);
        half(sa, sa + PA::BYTES, H0{});
        half(sa, sa + PA::BYTES, H1{});
        __syncthreads();
    }
    O::template tile<BM, BN, WM, WN, sizeof(smem)>(ep, t, g.N, acc, smem, wave, lane, early);
}

// ---------------------------------------------------------------- 256 x 256 tile

// 256 x 256, eight waves of 128 x 64, as mma16_kernel's: a stage is four phases of 16 matrix
// instructions, fragments and loads of later stages spread among them.
//   phase 0  half 0, block rows 0-3   reads half 1's A 0-3 and B; (three A slots) loads A of kt+2
//   phase 1  half 0, block rows 4-7   reads half 1's A 4-7
//   phase 2  half 1, block rows 0-3   then waits for stage kt+1, barrier
//   phase 3  half 1, block rows 4-7   reads half 0 of stage kt+1; loads the rest of kt+2
// bf16: three A slots and two B slots, all of the LDS; MXFP4: two of each and the scales.
// A full round's stage, 2048 cycles of matrix instructions on each SIMD, takes 1.39 us (bf16) or
// 1.76 us (MXFP4, four times the k): m x n x k 8192 x 4096 x 8192 367 and 130 us (1.50 and 4.2
// PFLOP/s); prologue, epilogue and launch take 7 to 9 us.  bf16 is bound by the matrix cores, 0.8 of them
// at the 1.8 GHz that the power limit leaves.  MXFP4 is not: at 2.08 GHz a stage is 3660 cycles,
// of which the scales' LDS reads, waits and lane swaps at its end, and eight loads and twelve
// fragment reads in one phase, take their part.
template <bool MX>
struct RaggedBigLds {
    static constexpr int NSA = MX ? 2 : 3, NSB = 2, OP = 256 * 128;
    static constexpr int B = NSA * OP, SCALES = B + NSB * OP;
    static constexpr int BYTES = SCALES + (MX ? 2 * ScalePanel<256, 256>::SLOT : 0);
};

template <bool MX, bool AT, bool BT, typename O>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void ragged_big_kernel(const RaggedArgs g, const typename O::Params ep) {
    constexpr int BM = 256, BN = 256, WM = 2, WN = 4, WTM = 128, WTN = 64, TM = 8, TN = 4;
    using L = RaggedBigLds<MX>;
    using PA = Panel<AT, BM, 8>;
    using PB = Panel<BT, BN, 8>;
    using SP = ScalePanel<BM, BN>;
    constexpr int LPA = PA::LP, LPB = PB::LP;
    constexpr bool A3 = L::NSA == 3;
    static_assert(L::BYTES <= 160 * 1024 && LPA == 4 && LPB == 4, "LDS");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    RaggedTile t;
    if (!ragged_tile<MX, AT, BT, BM, BN, true>(g, lane, t)) return;

    PA A;
    PB B;
    A.init(t.a, g.lda, t.rows, t.k, t.rows * 2, wave, lane);
    B.init(t.b, g.ldb, t.cols, BT && !AT ? g.K : t.k, t.cols * 2, wave, lane);
    SP S;
    if constexpr (MX) S.init(g, t, smem + L::SCALES, nullptr, wave, lane);
    const int nb = (g.K + 31) / 32;

    Frag<AT, BM> fa;
    Frag<BT, BN> fb;
    fa.init(lane, wm * WTM);
    fb.init(lane, wn * WTN);
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{};
    v4i af[2][TM], bf[2][TN];
    ScaleQuad xa[TM / 4], xb[1];

    auto mfma_rows = [&](auto hh, int r0) {
        constexpr int SS = decltype(hh)::value;
#pragma unroll
        for (int i = r0; i < r0 + TM / 2; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = MX ? mx_half<SS>(bf[SS][j], af[SS][i], acc[i][j], xb[0], xa[i / 4], i, j)
                               : bf_step(bf[SS][j], af[SS][i], acc[i][j]);
    };
    // A fragments [alo, alo + na) and (wb) the B fragments of half ss, with nl loads spread
    // among them.
    auto ops = [&](const uint8_t *sa, const uint8_t *sb, auto ss, int alo, auto na, auto wb, auto nl,
                   auto ld) {
        constexpr int SS = decltype(ss)::value, NA = decltype(na)::value;
        constexpr int NB = decltype(wb)::value ? TN : 0, NR = NA + NB, NL = decltype(nl)::value;
        int l = 0;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            // A[alo], B, then A[alo+1 ..]: the next phase's first products pair A[alo]
            // with every B fragment
            const int ra = r == 0 ? 0 : (r <= NB ? -1 : r - NB);
            if (ra >= 0) af[SS][alo + ra] = fa.read(sa, alo + ra, SS);
            else bf[SS][r - 1] = fb.read(sb, r - 1, SS);
            if ((r + 1) * NL / NR != r * NL / NR) ld(l++);
        }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using H = std::integral_constant<int, TM / 2>;
    using FA = std::integral_constant<int, TM>;
    constexpr int RA = AT ? 2 : 1, RB = BT ? 2 : 1;  // LDS reads per fragment
    constexpr int NM = (TM / 2) * TN, SPAN = NM * 7 / 8;

    auto a_slot = [&](int s) { return smem + s * L::OP; };
    auto b_slot = [&](int s) { return smem + L::B + s * L::OP; };
    auto scales = [&](int kt, int par) {  // of stage kt, which has landed
        const uint8_t *sc = smem + L::SCALES + ((kt >> 1) & 1) * SP::SLOT + par * 8;
        read_scales<TM / 4, WTM>(sc, wm * WTM, nb - kt * 8, lane, xa);
        read_scales<1, WTN>(sc, SP::A_ROWS + wn * WTN, nb - kt * 8, lane, xb);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if constexpr (MX) {
            if (s == 0) S.load(0);
        }
#pragma unroll
        for (int i = 0; i < LPA; ++i) A.load(a_slot(s), nullptr, i);
        A.next();
#pragma unroll
        for (int i = 0; i < LPB; ++i) B.load(b_slot(s), nullptr, i);
        B.next();
    }
    typename O::template EarlyTile<BM, BN, WM, WN> early;
    early.load(ep, t, g.N, wave, lane);
    wait_vmcnt<LPA + LPB>();
    stage_barrier();
    ops(a_slot(0), b_slot(0), I0{}, 0, FA{}, std::true_type{}, I0{}, [](int) {});
    if constexpr (MX) scales(0, 0);

    // Loads of stage kt+2 in phase 0 (L0, A's) and in phase 3 (L3, A's first).  The scales of
    // stages kt+2 and kt+3 go out in phase 3 of even stages.
    constexpr int L0 = A3 ? LPA : 0, L3 = LPA + LPB - L0;
    auto load3 = [&](int i, uint8_t *wa, uint8_t *wb) {
        if (!A3 && i < LPA) A.load(wa, nullptr, i);
        else B.load(wb, nullptr, i - (A3 ? 0 : LPA));
    };
    // A stage in two parts, up to its barrier and behind it: within each, the slots that are
    // loaded (wa, wb: stage kt+2's) and those that are read differ, and `restrict` says so
    // (see ragged_kernel).  No branches: they would end the scheduled block.
    auto before = [&](uint8_t *__restrict__ wa, const uint8_t *__restrict__ sa,
                      const uint8_t *__restrict__ sb) {
        mfma_rows(I0{}, 0);
        ops(sa, sb, I1{}, 0, H{}, std::true_type{}, std::integral_constant<int, L0>{},
            [&](int i) { A.load(wa, nullptr, i); });
        sched_ops<NM, TM / 2 * RA + TN * RB, L0, SPAN>();
        if constexpr (A3) A.next();
        mfma_rows(I0{}, TM / 2);
        ops(sa, sb, I1{}, TM / 2, H{}, std::false_type{}, I0{}, [](int) {});
        sched_ops<NM, TM / 2 * RA, 0, SPAN>();
        mfma_rows(I1{}, 0);
#pragma unroll
        for (int m = 0; m < NM; ++m) __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_barrier(0);  // (else these products move behind the barrier)
        wait_vmcnt<L0>();
        stage_barrier();
    };
    auto behind = [&](int kt, auto par, uint8_t *__restrict__ wa, uint8_t *__restrict__ wb,
                      const uint8_t *__restrict__ na, const uint8_t *__restrict__ nbp) {
#pragma unroll
        for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(af[1][i]));
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(bf[1][j]));
        mfma_rows(I1{}, TM / 2);
        if constexpr (MX && decltype(par)::value == 0) S.load(((kt >> 1) + 1) & 1);
        ops(na, nbp, I0{}, 0, FA{}, std::true_type{}, std::integral_constant<int, L3>{},
            [&](int i) { load3(i, wa, wb); });
        sched_ops<NM, TM * RA + TN * RB, L3, SPAN>();
        if constexpr (!A3) A.next();
        B.next();
        if constexpr (MX) scales(kt + 1, 1 - decltype(par)::value);
    };
    int s = 0;  // A slot of stage kt
    auto turn = [](int i) { return i == L::NSA - 1 ? 0 : i + 1; };
    auto step = [&](int kt, auto par) {
        constexpr int P = decltype(par)::value;
        const int s1 = turn(s), s2 = turn(s1);  // of kt+1 and kt+2
        before(a_slot(s2), a_slot(s), b_slot(P));
        behind(kt, par, a_slot(s2), b_slot(P), a_slot(s1), b_slot(1 - P));
        s = s1;
    };
    // A tile of at most half the rows: the lower waves only load, and the upper ones, one on
    // each SIMD, have the matrix cores to themselves.
    auto idle = [&](int kt, auto par) {
        constexpr int P = decltype(par)::value;
        const int s1 = turn(s);
        uint8_t *const wa = a_slot(turn(s1));
#pragma unroll
        for (int i = 0; i < L0; ++i) A.load(wa, nullptr, i);
        wait_vmcnt<L0>();
        stage_barrier();
        if constexpr (MX && P == 0) S.load(((kt >> 1) + 1) & 1);
#pragma unroll
        for (int i = 0; i < L3; ++i) load3(i, wa, b_slot(P));
        A.next();
        B.next();
        s = s1;
    };
    const int whole = MX && g.K % 32 ? t.KT - 1 : t.KT;  // stages without a cut block
    auto stages = [&](auto one) {
        for (int kt = 0; kt < whole; kt += 2) {
            one(kt, I0{});
            if (kt + 1 < whole) one(kt + 1, I1{});
        }
    };
    const bool idles = wm != 0 && t.rows <= WTM;
    if (!idles) stages(step);
    else stages(idle);
    wait_vmcnt<0>();
    __syncthreads();
    if (MX && whole < t.KT) {  // (its scales are in the registers, and half 0 uncut)
        mx_cut<BM>(a_slot(s), threadIdx.x, g.K);
        __syncthreads();
        if (!idles) {
            auto half = [&](auto hh) {
                ops(a_slot(s), b_slot(whole & 1), hh, 0, FA{}, std::true_type{}, I0{}, [](int) {});
                mfma_rows(hh, 0);
                mfma_rows(hh, TM / 2);
            };
            half(I0{});
            half(I1{});
        }
        __syncthreads();
    }
    O::template tile<BM, BN, WM, WN, sizeof(smem)>(ep, t, g.N, acc, smem, wave, lane, early);
}

// ---------------------------------------------------------------- few tiles

// Products with too few tiles to keep the CUs busy by themselves: the KS waves of a
// workgroup share one BM x BN tile and split K among them, stage kt to wave kt % KS.  Each
// wave fills its own ring of NS stages and waits for nothing but its own loads (no
// barriers); their sums are added in wave order through LDS at the end.  Bound by latency:
// 8x64x2048x1024 7.6 us (3.9 TB/s of the seven matrices that are used), 5.2 where the caches
// hold them from the call before.
template <bool MX, int BM, int BN, int KS, int NS>
struct RaggedWaveLds {
    static constexpr int STAGE = (BM + BN) * 128 + (MX ? 2048 : 0);  // operands, scales
    static constexpr int RING = KS * NS * STAGE, SUMS = KS * BM * (BN + 4) * 4;
    static constexpr int BYTES = RING > SUMS ? RING : SUMS;
};

template <bool MX, bool AT, bool BT, typename O, int BM, int BN, int KS, int NS, bool ONCE>
__global__ __launch_bounds__(KS * 64)
__attribute__((amdgpu_waves_per_eu(ragged_waves(RaggedWaveLds<MX, BM, BN, KS, NS>::BYTES, KS),
                                   ragged_waves(RaggedWaveLds<MX, BM, BN, KS, NS>::BYTES, KS))))
void ragged_wave_kernel(const RaggedArgs g, const typename O::Params ep) {
    constexpr int TM = BM / 16, TN = BN / 16, QA = (TM + 3) / 4, QB = (TN + 3) / 4;
    using L = RaggedWaveLds<MX, BM, BN, KS, NS>;
    using PA = Panel<AT, BM, 1>;
    using PB = Panel<BT, BN, 1, ONCE>;
    constexpr int LPW = PA::LP + PB::LP + (MX ? 2 : 0);
    static_assert(L::BYTES <= 160 * 1024 && (!MX || (BM <= 64 && BN <= 64)),
                  "LDS, one scale load per operand");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RaggedTile t;
    if (!ragged_tile<MX, AT, BT, BM, BN, false>(g, lane, t)) return;

    PA A;
    PB B;
    A.init(t.a, g.lda, t.rows, t.k, t.rows * 2, 0, lane);
    B.init(t.b, g.ldb, t.cols, BT && !AT ? g.K : t.k, t.cols * 2, 0, lane);
    A.skip(wave);
    B.skip(wave);
    // Scales: 16 bytes of every row, of stage kt and its neighbour kt ^ 1.
    const int nb = (g.K + 31) / 32;
    const uint8_t *sa = nullptr, *sb = nullptr;
    uint32_t va = 0, vb = 0;
    if constexpr (MX) {
        sa = uniform(g.sa + t.row0 * g.lsa);
        sb = uniform(g.sb + t.g * g.bssb + (int64_t)t.n0 * g.lsb);
        va = lane < t.rows ? (uint32_t)(lane * (int)g.lsa) : kOutOfRange;
        vb = lane < t.cols ? (uint32_t)(lane * (int)g.lsb) : kOutOfRange;
    }
    uint8_t *const ring = smem + wave * (NS * L::STAGE);
    auto load_stage = [&](int kt, uint8_t *d) {
#pragma unroll
        for (int i = 0; i < PA::LP; ++i) A.load(d, nullptr, i);
#pragma unroll
        for (int i = 0; i < PB::LP; ++i) B.load(d + PA::BYTES, nullptr, i);
        if constexpr (MX) {
            const uint32_t n = __builtin_amdgcn_readfirstlane(kt < t.KT ? kMaxRecords : 0);
            dma16(sa + kt / 2 * 16, n, va, d + PA::BYTES + PB::BYTES);
            dma16(sb + kt / 2 * 16, n, vb, d + PA::BYTES + PB::BYTES + 1024);
        }
        A.skip(KS);
        B.skip(KS);
    };

    Frag<AT, BM> fa;
    Frag<BT, BN> fb;
    fa.init(lane, 0);
    fb.init(lane, 0);
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{};

    auto products = [&](int kt, const uint8_t *s) {  // of stage kt, which has landed
        ScaleQuad xa[QA], xb[QB];
        if constexpr (MX) {
            const uint8_t *sc = s + PA::BYTES + PB::BYTES + (kt & 1) * 8;
            read_scales<QA, BM>(sc, 0, nb - kt * 8, lane, xa);
            read_scales<QB, BN>(sc + 1024, 0, nb - kt * 8, lane, xb);
        }
        auto half = [&](auto hh) {
            constexpr int SS = decltype(hh)::value;
            v4i af[TM], bf[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) bf[j] = fb.read(s + PA::BYTES, j, SS);
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = fa.read(s, i, SS);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[i][j] = MX ? mx_half<SS>(bf[j], af[i], acc[i][j], xb[j / 4], xa[i / 4], i, j)
                                   : bf_step(bf[j], af[i], acc[i][j]);
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
    };
    // (wr and sa differ: see ragged_kernel)
    auto kstep = [&](int kt, uint8_t *__restrict__ wr, const uint8_t *__restrict__ s) {
        wait_vmcnt<(NS - 2) * LPW>();
        asm volatile("" ::: "memory");  // (no access moves over the wait)
        load_stage(kt + (NS - 1) * KS, wr);
        products(kt, s);
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) load_stage(wave + i * KS, ring + i * L::STAGE);
    typename O::template EarlyWaves<BM, BN, KS> early;
    early.load(ep, t, g.N, wave, lane);
    int slot = 0, kt = wave;
    const int whole = MX && g.K % 32 ? t.KT - 1 : t.KT;  // stages without a cut block
    for (; kt < whole; kt += KS) {
        kstep(kt, ring + (slot == 0 ? NS - 1 : slot - 1) * L::STAGE, ring + slot * L::STAGE);
        slot = slot == NS - 1 ? 0 : slot + 1;
    }

    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (MX && kt < t.KT) {  // this wave's: its LDS accesses take effect in order
        mx_cut<BM>(ring + slot * L::STAGE, lane, g.K);
        asm volatile("" ::: "memory");
        products(kt, ring + slot * L::STAGE);
    }
    __syncthreads();
    O::template waves<BM, BN, KS, sizeof(smem)>(ep, t, g.N, acc, smem, wave, lane, early);
}

// ---------------------------------------------------------------- operands of any alignment

// Rows that miss the 16-byte alignment of the direct-to-LDS loads (an odd k or n) go
// through registers: 16-byte loads at any address, two stages ahead, written to the stage's
// slots.  Several workgroups on a CU, whose small rings leave the LDS room for, keep the
// loads in flight that a deep ring would.  Decoding reads 4x64x2830x3792's weights at 5.1 TB/s
// (16.8 us); a long product takes 1.6 times an aligned one's time (16384x8x2049x2047 246 us).
template <bool TR, int W, int NW>
struct RegPanel {
    static constexpr int BYTES = W * 128, NI = BYTES / 1024, LP = (NI + NW - 1) / NW;
    static constexpr int kNone = INT32_MAX;
    static constexpr bool CODES = false;
    using Reg = v4i;
    // 16 bytes before the next stage (a chunk across the end of a row is read back from that
    // end, which may lie before the stage's first byte).
    const uint8_t *base;
    int ld, left;      // row stride in bytes; contraction left: bytes, or rows (TR)
    uint32_t vo[LP];   // this lane's offsets from `base`
    int pos[LP];       // where they lie in the contraction, kNone: outside the tile
    int cut[TR ? LP : 1];  // TR: bytes of the chunk past the matrix's columns
    int wave, lane;

    // lim: rows of the tile; TR: bytes of its columns that are in the matrix
    __device__ __forceinline__ void init(const uint8_t *b, int64_t ld_, int k, int lim, int wave_,
                                         int lane_) {
        base = uniform(b) - 16;
        ld = (int)ld_;
        left = k;
        wave = wave_;
        lane = lane_;
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            const int at = (wave * LP + i) * 64 + lane;  // 16-byte slot of the stage
            if constexpr (TR) {
                const int row = at / (W / 8), slot = at % (W / 8);
                const int ch = ((((slot >> 1) ^ tr_unit<W>(row)) << 1) | (slot & 1)) * 16;
                cut[i] = lim - ch < 16 ? 16 - (lim - ch) : 0;
                vo[i] = (uint32_t)(16 + row * ld + ch - cut[i]);
                pos[i] = mine(i) && ch < lim ? row : kNone;
            } else {
                const int row = at / 8, ch = ((at % 8) ^ swz_of<128>(row)) * 16;
                vo[i] = (uint32_t)(16 + row * ld + ch);
                pos[i] = mine(i) && row < lim ? ch : kNone;
            }
        }
    }
    __device__ __forceinline__ bool mine(int i) const { return NI % NW == 0 || wave * LP + i < NI; }
    // A chunk's last 16 - c bytes, moved to its beginning (c: 2 .. 14).
    __device__ __forceinline__ static v4i shifted(v4i v, int c) {
        typedef uint64_t v2l __attribute__((ext_vector_type(2)));
        v2l w = __builtin_bit_cast(v2l, v);
        const int s = c * 8;
        w[0] = s >= 64 ? w[1] >> (s - 64) : w[0] >> s | w[1] << (64 - s);
        w[1] = s >= 64 ? 0 : w[1] >> s;
        return __builtin_bit_cast(v4i, w);
    }
    __device__ __forceinline__ void load(v4i (&r)[LP]) {
        typedef int v4i_any2 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
        for (int i = 0; i < LP; ++i) {
            v4i v = {};
            if constexpr (TR) {
                if (pos[i] < left) {
                    v = *(const v4i_any2 *)(base + vo[i]);
                    if (cut[i]) v = shifted(v, cut[i]);
                }
            } else if (pos[i] < left) {
                const int c = left - pos[i] < 16 ? 16 - (left - pos[i]) : 0;
                v = *(const v4i_any2 *)(base + (vo[i] - (uint32_t)c));
                if (c) v = shifted(v, c);
            }
            r[i] = v;
        }
    }
    __device__ __forceinline__ void skip(int stages) {
        base += TR ? (int64_t)stages * 64 * ld : stages * 128;
        left -= stages * (TR ? 64 : 128);
    }
    __device__ __forceinline__ void store(const v4i (&r)[LP], uint8_t *dst) const {
#pragma unroll
        for (int i = 0; i < LP; ++i)
            if (mine(i)) *(v4i *)(dst + (wave * LP + i) * 1024 + lane * 16) = r[i];
    }
};

// LEFT: A's panel, with RegPanel's members.
template <bool AT, bool BT, typename O, int BM, int BN, int WM, int WN,
          typename LEFT = RegPanel<AT, BM, WM * WN>>
__global__ __launch_bounds__(WM * WN * 64)
void ragged_reg_kernel(const RaggedArgs g, const typename O::Params ep) {
    constexpr int NW = WM * WN;
    constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    using PA = LEFT;
    using PB = RegPanel<BT, BN, NW>;
    constexpr int STAGE = PA::BYTES + PB::BYTES, SUMS = NW * 16 * (WTN + 4) * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE > SUMS ? 2 * STAGE : SUMS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    RaggedTile t;
    if (!ragged_tile<false, AT, BT, BM, BN, false>(g, lane, t)) return;
    // (t.k is rounded up to 16 bytes, for rows that are padded)
    const int kb = AT ? t.k : g.K * 2;
    PA A;
    PB B;
    if constexpr (PA::CODES) A.init(g, t, wave, lane);
    else A.init(t.a, g.lda, kb, AT ? t.rows * 2 : t.rows, wave, lane);
    B.init(t.b, g.ldb, BT && !AT ? g.K : kb, BT ? t.cols * 2 : t.cols, wave, lane);

    Frag<AT, BM> fa;
    Frag<BT, BN> fb;
    fa.init(lane, wm * WTM);
    fb.init(lane, wn * WTN);
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{};

    typename PA::Reg ra[2][PA::LP];
    v4i rb[2][PB::LP];
    auto get = [&](int set) __attribute__((always_inline)) {
        A.load(ra[set]);
        B.load(rb[set]);
        A.skip(1);
        B.skip(1);
    };
    auto put = [&](int set, uint8_t *d) __attribute__((always_inline)) {
        A.store(ra[set], d);
        B.store(rb[set], d + PA::BYTES);
        get(set);
    };
    // Stage kt from slot PAR; stage kt+1, in registers, goes to the other one, and the loads
    // of stage kt+3 take its registers.
    auto kstep = [&](auto par) __attribute__((always_inline)) {
        constexpr int PAR = decltype(par)::value;
        const uint8_t *const sa = smem + PAR * STAGE, *const sb = sa + PA::BYTES;
        put(1 - PAR, smem + (1 - PAR) * STAGE);
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
            v4i af[TM], bf[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) bf[j] = fb.read(sb, j, ss);
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = fa.read(sa, i, ss);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = bf_step(bf[j], af[i], acc[i][j]);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's writes and reads
        stage_barrier();
    };
    get(0);
    get(1);
    typename O::template EarlyTile<BM, BN, WM, WN> early;
    early.load(ep, t, g.N, wave, lane);
    put(0, smem);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    stage_barrier();
    for (int kt = 0; kt < t.KT; kt += 2) {
        kstep(std::integral_constant<int, 0>{});
        if (kt + 1 < t.KT) kstep(std::integral_constant<int, 1>{});
    }
    __syncthreads();
    O::template tile<BM, BN, WM, WN, sizeof(smem)>(ep, t, g.N, acc, smem, wave, lane, early);
}

// The same with K split over the KS waves of a workgroup (see ragged_wave_kernel): a wave's
// stages go through a slot of its own, so it waits for its own loads only.
template <bool AT, bool BT, typename O, int BM, int BN, int KS>
__global__ __launch_bounds__(KS * 64)
void ragged_reg_wave_kernel(const RaggedArgs g, const typename O::Params ep) {
    constexpr int TM = BM / 16, TN = BN / 16;
    using PA = RegPanel<AT, BM, 1>;
    using PB = RegPanel<BT, BN, 1>;
    constexpr int STAGE = PA::BYTES + PB::BYTES, SUMS = KS * BM * (BN + 4) * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KS * STAGE > SUMS ? KS * STAGE : SUMS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RaggedTile t;
    if (!ragged_tile<false, AT, BT, BM, BN, false>(g, lane, t)) return;
    const int kb = AT ? t.k : g.K * 2;
    PA A;
    PB B;
    A.init(t.a, g.lda, kb, AT ? t.rows * 2 : t.rows, 0, lane);
    B.init(t.b, g.ldb, BT && !AT ? g.K : kb, BT ? t.cols * 2 : t.cols, 0, lane);
    A.skip(wave);
    B.skip(wave);
    uint8_t *const sa = smem + wave * STAGE, *const sb = sa + PA::BYTES;

    Frag<AT, BM> fa;
    Frag<BT, BN> fb;
    fa.init(lane, 0);
    fb.init(lane, 0);
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{};
    v4i ra[2][PA::LP], rb[2][PB::LP];
    auto get = [&](int set) {
        A.load(ra[set]);
        B.load(rb[set]);
        A.skip(KS);
        B.skip(KS);
    };
    auto kstep = [&](auto par) {
        constexpr int PAR = decltype(par)::value;
        A.store(ra[PAR], sa);
        B.store(rb[PAR], sb);
        get(PAR);
        asm volatile("" ::: "memory");  // (a wave's LDS accesses take effect in order)
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
            v4i af[TM], bf[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) bf[j] = fb.read(sb, j, ss);
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = fa.read(sa, i, ss);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = bf_step(bf[j], af[i], acc[i][j]);
        }
        asm volatile("" ::: "memory");
    };
    get(0);
    get(1);
    typename O::template EarlyWaves<BM, BN, KS> early;
    early.load(ep, t, g.N, wave, lane);
    for (int kt = wave; kt < t.KT; kt += 2 * KS) {
        kstep(std::integral_constant<int, 0>{});
        if (kt + KS < t.KT) kstep(std::integral_constant<int, 1>{});
    }
    __syncthreads();
    O::template waves<BM, BN, KS, sizeof(smem)>(ep, t, g.N, acc, smem, wave, lane, early);
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

// The kernels' tile shapes.
// ring: BM x BN on WM x WN waves, NS stages; big: 256 x 256; wave: BM x BN, K split over KS
// waves.  ONCE: B nontemporally.
template <int BM_, int BN_, int WM_, int WN_, int NS_, bool ONCE_ = false>
struct RingTile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, KIND = 0;
    static constexpr bool ONCE = ONCE_;
};
struct BigTile {
    static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, NS = 0, KIND = 1;
    static constexpr bool ONCE = false;
};
template <int BM_, int BN_, int KS, int NS_, bool ONCE_ = false>
struct WaveTile {
    static constexpr int BM = BM_, BN = BN_, WM = 1, WN = KS, NS = NS_, KIND = 2;
    static constexpr bool ONCE = ONCE_;
};

// reg: operands of any alignment.
template <int BM_, int BN_, int WM_, int WN_>
struct RegTile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = 0, KIND = 3;
    static constexpr bool ONCE = false;
};

template <int BM_, int BN_, int KS>
struct RegWaveTile {
    static constexpr int BM = BM_, BN = BN_, WM = 1, WN = KS, NS = 0, KIND = 4;
    static constexpr bool ONCE = false;
};

template <bool MX, bool AT, bool BT, typename O, typename T>
static hipError_t ragged_go(const RaggedArgs &g, const typename O::Params &ep, hipStream_t stream) {
    constexpr int BM = T::BM, BN = T::BN;
    // 32-bit offsets inside a panel, with the loads of rows past its edge
    const int64_t kbytes = MX ? (int64_t)(g.K + 31) / 32 * 16 : (int64_t)g.K * 2;
    if ((AT ? 64 : BM) * g.lda + kbytes > (int64_t)kMaxRecords ||
        (BT ? 64 * g.ldb + BN * 2 : BN * g.ldb + kbytes) > (int64_t)kMaxRecords ||
        (MX && 64 * (g.lsa > g.lsb ? g.lsa : g.lsb) > (int64_t)kMaxRecords))
        return hipErrorInvalidValue;
    const int64_t per =
        (int64_t)((g.K + BM - 1) / BM) * ((g.N + BN - 1) / BN) * (AT ? g.splits : 1);
    if (AT && per > INT32_MAX - 8) return hipErrorInvalidValue;
    const int64_t tiles = AT ? (int64_t)g.G * wgrad_share((int)per) * 8
                             : ragged_tiles(g, BM, BN) + (T::KIND == 1 ? g.cus : 8);
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid = ragged_grid(tiles), block(T::WM * T::WN * 64);
    if constexpr (T::KIND == 1)
        hipLaunchKernelGGL((ragged_big_kernel<MX, AT, BT, O>), grid, block, 0, stream, g, ep);
    else if constexpr (T::KIND == 2)
        hipLaunchKernelGGL((ragged_wave_kernel<MX, AT, BT, O, BM, BN, T::WN, T::NS, T::ONCE>), grid, block, 0,
                           stream, g, ep);
    else if constexpr (T::KIND == 3)
        hipLaunchKernelGGL((ragged_reg_kernel<AT, BT, O, BM, BN, T::WM, T::WN>), grid, block, 0,
                           stream, g, ep);
    else if constexpr (T::KIND == 4)
        hipLaunchKernelGGL((ragged_reg_wave_kernel<AT, BT, O, BM, BN, T::WN>), grid, block, 0, stream,
                           g, ep);
    else
        hipLaunchKernelGGL((ragged_kernel<MX, AT, BT, O, BM, BN, T::WM, T::WN, T::NS, T::ONCE>), grid,
                           block, 0, stream, g, ep);
    return hipGetLastError();
}

// Tiles of a forward product whose groups are alike.
inline int64_t even_tiles(const RaggedArgs &g, int64_t avg, int bm, int bn) {
    const int64_t groups = g.off ? (g.G < g.M ? g.G : g.M) : 1;
    return groups * ((avg + bm - 1) / bm) * (((int64_t)g.N + bn - 1) / bn);
}

// Expected time in us of a forward product with more than 16 rows a group on a BM x BN tile:
//   2 + sqrt(c^2 + m^2),  c = (a + b*stages) * (1 + h*(y' - 1)),  m = bytes / bw
// with y tiles per CU (a group's last tile half full on average), y' = q*ceil(y) + (1-q)*y, at
// least 1.  The constants are the least-squares fit of log times of 110 products x 3 operand
// kinds (17..4096 rows a group, 1..128 groups, k and n 128..8192, graph-timed with rotating
// weights); the tile they pick took 1.009 (bf16) and 1.011 (MXFP4) times the fastest of the seven
// in the geometric mean, 1.31 at worst.  The seven are those of 13 shapes that leave the least
// behind the fastest of all (1.02).
struct RaggedCost {
    int bm, bn;
    double a, b, h, bw, q;
};
constexpr RaggedCost kRaggedCost[2][7] = {
    {{64, 64, 0.91, 0.287, 0.97, 4.29, 0.55},     // bf16
     {64, 128, 1.26, 0.403, 0.99, 4.69, 0.67},
     {128, 128, 1.84, 0.492, 1.31, 4.98, 0.96},
     {128, 256, 2.72, 0.794, 1.29, 4.97, 0.79},
     {256, 256, 4.25, 0.901, 1.17, 3.65, 1.00},
     {32, 64, 1.52, 0.156, 1.28, 3.86, 0.96},
     {16, 32, 1.04, 0.095, 0.86, 3.50, 0.87}},
    {{64, 64, 1.64, 0.408, 0.74, 4.30, 0.58},     // MXFP4
     {64, 128, 1.99, 0.549, 0.75, 4.53, 0.62},
     {128, 128, 2.22, 0.755, 0.83, 4.61, 0.50},
     {128, 256, 3.49, 1.051, 1.17, 4.72, 1.00},
     {256, 256, 5.22, 1.164, 1.17, 3.24, 1.00},
     {32, 64, 1.93, 0.162, 1.24, 3.26, 0.91},
     {16, 32, 1.87, 0.086, 1.08, 3.10, 0.88}}};

inline double ragged_cost(const RaggedCost &c, const RaggedArgs &g, int64_t groups, int64_t avg,
                          int64_t kbytes) {
    const double tm = groups == 1 ? (double)((avg + c.bm - 1) / c.bm)
                                  : std::max(1.0, (double)avg / c.bm + 0.5);
    const double y = groups * tm * (double)((g.N + c.bn - 1) / c.bn) / std::max(g.cus, 1);
    const double rounds = std::max(1.0, c.q * std::ceil(y) + (1.0 - c.q) * y);
    const double work = (c.a + c.b * (double)((kbytes + 127) / 128)) * (1.0 + c.h * (rounds - 1.0));
    const double bytes = ((double)groups * g.N + g.M) * (double)kbytes + 2.0 * g.M * g.N;
    const double mem = bytes / (c.bw * 1e6);
    return 2.0 + std::sqrt(work * work + mem * mem);
}

// The cheapest of the seven for a product of more than 16 rows a group, and its time.
template <bool MX>
inline int ragged_best(const RaggedArgs &g, int64_t groups, int64_t avg, int64_t kbytes,
                       double *cost) {
    int best = 0;
    for (int i = 0; i < 7; ++i) {
        const double c = ragged_cost(kRaggedCost[MX ? 1 : 0][i], g, groups, avg, kbytes);
        if (i == 0 || c < *cost) {
            best = i;
            *cost = c;
        }
    }
    return best;
}

// Expected time in us of a weight gradient, or of a product of operands of any alignment, on
// one tile shape: y tiles per CU, each of `stages` stages, over `bytes` of operands and output.
//   2 + sqrt((a + b*stages + (c1 + c2*stages)*(y' - 1))^2 + (bytes / bw)^2)
// with y' = q*ceil(y) + (1-q)*y, at least 1: the first tile of a CU takes its latency, and
// several workgroups on a CU overlap those after it.
struct TileTime {
    int bm, bn;
    double a, b, c1, c2, bw, q;
};

inline double tile_time(const TileTime &c, double y, double stages, double bytes) {
    const double rounds = std::max(1.0, c.q * std::ceil(y - 1e-9) + (1.0 - c.q) * y);
    const double work = c.a + c.b * stages + (c.c1 + c.c2 * stages) * (rounds - 1.0);
    const double mem = bytes / (c.bw * 1e6);
    return 2.0 + std::sqrt(work * work + mem * mem);
}

// f(the tile of a forward product), by the average rows of a group (the host does not know
// more).  Times in us, graph-timed with rotating weights on one card, as rows x groups x k x n
// with k-contiguous / n-contiguous bf16 / MXFP4 weights.  For up to 16 rows a group the
// rules below took 1.08 / 1.12 / 1.05 times the fastest of 9 to 13 tiles in the geometric mean
// (103 products, 1..128 groups, k and n 128..8192; 1.45 at worst), and 1.12 / 1.13 / 1.08 where
// one group has eight ninths of the rows (47 products; 1.71 at worst: tiles follow the average
// group, and that one reads its weights again every 16 rows).
template <bool MX, bool BT, typename F>
static auto forward_tile(const RaggedArgs &g, F f) {
#define GK_GO(...) return f(__VA_ARGS__{})
#define GK_GO_ONCE(...) \
    do { \
        if (once) GK_GO(__VA_ARGS__, true>); \
        GK_GO(__VA_ARGS__>); \
    } while (0)
    const int64_t cus = g.cus;
    const int64_t groups = g.off ? (g.G < g.M ? g.G : g.M) : 1;
    const int64_t avg = (g.M + groups - 1) / groups;
    const int64_t kbytes = MX ? (int64_t)g.K / 2 : (int64_t)g.K * 2, stages = (kbytes + 127) / 128;
    // Weights that tiles of 64 rows read once, and that would fill half of the 256 MB
    // Infinity Cache, go past it: on the tiles picked 64x32x2048x4096 takes 72.4 / 70.9 / 23.8
    // through it and 64.4 / 63.8 / 21.9 past it, 16x8x4096x11008 111 / 120 / 32.7 and
    // 97 / 110 / 30.6.  Smaller ones stay there from one call to the next, and are read again
    // by every further tile: 150x3x2048x2048 on 64 x 128 13.7 / 14.4 / 8.0 through it, 17.8 /
    // 18.3 / 8.2 past it.
    const bool once = avg <= 64 && groups * g.N * kbytes >= (int64_t(128) << 20);
    if (avg <= 16) {
        // One 16-row tile per group: the weights are read once, HBM-bound.  Where K is split
        // over the waves nothing waits at barriers and a few tiles keep many loads in
        // flight: 8x64x2048x1024 7.6 / 9.0 / 5.1 against 9.5 / 8.8 / 6.4 on the ring,
        // 64x32x2048x4096 64 / 94 / 44 against 66 / 70 / 22.  It reads 64-byte pieces
        // of n-contiguous rows (32 columns) and a scale load per stage, so those two
        // layouts take it for few tiles only, and k of few stages never (128x100x512x600
        // 15.1 / 15.3 / 17.2 against 10.5 / 11.0 / 6.8).
        const int64_t few = even_tiles(g, avg, 16, 64);
        if (stages >= 8 && (MX ? few <= cus / 2 : BT ? few <= cus / 4 : stages >= 16)) {
            GK_GO_ONCE(WaveTile<16, 32, 4, 3);
        }
        // Up to a tile per CU: MXFP4 in 64-row pieces of the weights, split alike: 8x1x4096x14336
        // 8.3 against 9.5 on the ring, 64x16x4096x896 8.0 / 9.4 (16 x 32: 10.0); n-contiguous
        // weights do not gain (8x2x4096x8192 29.1 / 27.7).
        if constexpr (MX) {
            if (stages >= 8 && few <= cus) GK_GO_ONCE(WaveTile<16, 64, 4, 2);
        }
        // Up to two: 128 columns instead, which a CU reads in longer pieces and in one tile:
        // - / 15.7 / 6.6 against - / 21.5 / 7.3 (12x12x1536x2560), - / 34.4 / 11.2 against
        // - / 42.8 / 12.4 (8x4x4096x5120); k-contiguous ones do not gain (39.5 / 33.3).  Where
        // uneven groups of more rows need second tiles beyond those, 64 rows hold them:
        // 64x8x4096x4096 - / 42 / 16.4 against - / 62 / 23.8.
        // Many tiles: n-contiguous rows in 256-byte pieces, MXFP4 tiles of 8 rows and more:
        // 64x32x2048x4096 - / 64 against - / 70, 256x32x2048x2048 - / 44 / 17.1 against
        // - / 48 / 18.7; 8x1x4096x14336 - / 35 / 12.0 against - / 26 / 9.5 (too few)
        if constexpr (MX || BT) {
            const bool two = few > cus && few <= 2 * cus;
            if (two && (avg <= 4 || 2 * few <= 3 * cus)) GK_GO_ONCE(RingTile<16, 128, 1, 4, 4);
            if (two || ((BT || avg > 4) && even_tiles(g, avg, 64, 128) >= 2 * cus))
                GK_GO_ONCE(RingTile<64, 128, 2, 2, 3);
        }
        GK_GO_ONCE(RingTile<16, 64, 1, 4, 4);
    }
    double cost = 0;
    switch (ragged_best<MX>(g, groups, avg, kbytes, &cost)) {
    case 1: GK_GO_ONCE(RingTile<64, 128, 2, 2, 3);
    case 2: GK_GO_ONCE(RingTile<128, 128, 2, 4, MX ? 2 : 4);
    case 3: GK_GO(RingTile<128, 256, 2, 4, 3>);
    case 4: GK_GO(BigTile);
    case 5: GK_GO(WaveTile<32, 64, 4, 2>);
    case 6: GK_GO(WaveTile<16, 32, 4, 3>);
    default: GK_GO_ONCE(RingTile<64, 64, 2, 2, 4);
    }
#undef GK_GO_ONCE
#undef GK_GO
}

// f(the tile of a forward product of operands of any alignment) that grouped_plan_any chose.
template <typename F>
static auto any_align_tile(const RaggedArgs &g, F f) {
    switch (g.tile) {
    case 0: return f(RegTile<128, 128, 2, 4>{});
    case 1: return f(RegTile<128, 64, 4, 2>{});
    case 2: return f(RegTile<32, 64, 1, 4>{});
    case 3: return f(RegWaveTile<16, 32, 4>{});
    default: return f(RegWaveTile<16, 32, 8>{});
    }
}

template <bool MX, bool BT, EpiKind E>
static hipError_t ragged_forward(const RaggedArgs &g, const EpiParams &ep, hipStream_t stream) {
    return forward_tile<MX, BT>(
        g, [&](auto t) { return ragged_go<MX, false, BT, PlainOut<E>, decltype(t)>(g, ep, stream); });
}

template <typename T>
RaggedPlan plan_of(T) {
    return RaggedPlan{T::KIND, T::BM, T::BN, T::KIND == 2 || T::KIND == 4 ? T::WN : 1, T::ONCE};
}

}  // namespace gk
