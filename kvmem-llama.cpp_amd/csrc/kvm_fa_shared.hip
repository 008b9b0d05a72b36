// kvm_fa_shared.hip -- decode / verify attention of several conversations that share a
// long prefix (kvm_fa_decode_shared): every query attends over the prefix window's cells
// and its own conversation's, one softmax over both.
//
//   o_t = sum_c p_tc v_c / sum_c p_tc, p_tc = exp(scale q_t . k_c - m_t) over the cells c of
//   both windows with 0 <= position <= the query's
//
// splits over any parts of the cells into (m, l, o) of each part, joined by the parts'
// maxima.  A part is a piece: some tiles of one window for a unit, 32 or 128 rows of a kv
// head (a row is a token and a query head of the group).  The prefix's rows are all
// conversations' tokens side by side, so its keys and values are read, and brought to f16,
// once for a unit's rows; a conversation's own window has that conversation's rows.
// k_fs_wide and k_fs_narrow form the pieces, k_fs_join joins those of each row.
//
// S^T = K Q^T and O^T += V^T P^T on 32x32x16 f16 MFMAs, 32 rows a wave.  Quantised tiles
// become f16 on the way: K and V as (f16)(q d); Q and P are rounded to f16, as the products take
// them, everything else is fp32.  (fp32 outputs are 1.8e-4 - 3.9e-4 from the 64-bit ones, 2-norm; bf16
// ones 1.7e-3, their own rounding.)  Key order: score row i of a half tile is key i with bits 2 and 3
// swapped, so that a lane's scores are 8 consecutive keys of each 16, what the P V operand wants.
//   narrow units (quantised windows of few rows): workgroups of 4 waves, two a CU.
//     Each wave takes every fourth half of the piece's tiles.  Nothing is shared in the loop and no
//     barrier is in it: tiles go from memory into registers (the tile layout is the matrix
//     operands') and are converted there; the waves' sums meet in LDS at the end.
//   wide units: workgroups of 8 waves, one a CU.  Waves 0 - 3 have 32 rows each and take every
//     key; waves 4 - 7 bring the next tile into one of two LDS buffers, converted, while the
//     other is worked on.
// A value that f16 does not hold as a finite number is taken out of tiles that some row does not see
// (fs_clear) and added in fp32 to the rows that do (fs_add_odd).  In other tiles nothing looks for one:
// where a piece's sums come out as no finite numbers, it is formed again with every tile treated so
// (CAREFUL), which finite values, and infinite ones under a p that f16 rounds to 0, then come out of right.
// (Looking costs 0.2 us of 8.3 and 0.4 of 24.5 over f16 windows, nothing measurable over others.)
// A workgroup has one piece: the units of a window are cut into equal numbers of pieces, and
// longer ones into more.  The tiles are taken in an order that steps through a window in
// strides: a part-filled window's live tiles are spread evenly over its pieces.
#include "kvm_f16_dev.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#define FS_LANES 64u             // conversations of a call
#define FS_SEGS (FS_LANES + 1)   // windows: theirs and the prefix
#define FS_BATCH 256u            // tiles of a piece that are looked at at a time
#define FS_LAZY 8.0f             // log2 growth of a row's maximum tolerated before a rescale

typedef float kvm_f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *fs_lds_ptr;
typedef float kvm_f32x2 __attribute__((ext_vector_type(2)));

// A window with the rows that attend over it.
struct fs_seg {
    const uint8_t *k, *v;
    const int32_t *cell_pos;
    uint32_t n_tiles, mult;      // tile i of a unit's order is (i mult) mod n_tiles
    uint32_t row0, n_rows;       // rows [row0, row0 + n_rows) of every kv head
    uint32_t step;               // from tile i to tile i + 4 times the waves of a workgroup (mod n_tiles)
    uint32_t pieces, per, more;  // of a unit: pieces of `per` tiles, the first `more` of one more
};

struct fs_args {
    const void *q;
    const int32_t *q_pos;
    float *ws_o;                 // pieces of 32 rows: [slot][dim / 8][lane][4]
    float *ws_ml;                // [slot][row][2]: scaled maximum, sum
    uint32_t H, G, n_head, n_rows;
    uint32_t wide, narrow;       // pieces; the wide ones' segments come first
    float c, q_sign;             // |scale| log2(e); q times -1 for a negative scale, and 0 (c = 1) for none
    int q_type;
    float inv_g;                 // 1 / G
    // Pieces of the segments before; a segment's: [head][piece of the unit][unit of the head],
    // so that neighbours read the same tiles.  A wide piece has 4 slots, a narrow one 1.
    uint32_t piece0[FS_SEGS];    // (past the last segment: ~0)
    fs_seg seg[FS_SEGS];
};
static_assert(sizeof(fs_args) <= 4096, "kernel arguments");

// What the join reads.
struct fs_join_args {
    const float *ws_o, *ws_ml;
    void *out;
    int out_type;
    uint32_t G, n_head, n_rows;
    uint32_t pre_pieces, pre_wide;                        // a prefix unit's (none: no prefix)
    // conversations with a window, in order: first row (the rest: ~0), rows, pieces of a unit
    // (bit 31: wide), first slot
    uint32_t row0[FS_LANES], rows[FS_LANES], pieces[FS_LANES], slot0[FS_LANES];
};

__host__ __device__ inline uint32_t fs_unit_rows(bool wide) { return wide ? 128u : 32u; }
__host__ __device__ inline uint32_t fs_row_tiles(bool wide, uint32_t n_rows) { return (n_rows + fs_unit_rows(wide) - 1) / fs_unit_rows(wide); }

template <int D, bool QUANT>
struct fs_geo {
    static constexpr int KS = D / 16, NB = D / 32, DT = D / 32;              // k-steps, 32-dim blocks, dim tiles
    static constexpr uint32_t KB = QUANT ? 64u * D + 128u * NB : 128u * D, VB = QUANT ? 32u * D + 128u * NB : 128u * D;
    static constexpr uint32_t TB = 128u * D;              // bytes of an f16 K (or V) tile
    static constexpr uint32_t QU = 528;                   // LDS bytes of a unit of Q: 8 dims of 32 rows, 16 bytes apart in the banks
    // Of 256 dims every third Q operand of a wide unit is read from LDS: all 16 in registers
    // are 24 too many (spilled, their reloads were half of a tile's time)
    static constexpr int QL = D == 256 ? 5 : 0;
    static constexpr int SETS = D == 256 ? 1 : 2;         // half tiles that a wave has in registers
    static constexpr int NQ = D / 32;                     // quads that a wave adds up at the end of a narrow piece
};

// What both kinds have in LDS; NW: waves.
template <int D, int NW>
struct fs_list {
    alignas(16) float odd_v[4][D];
    uint32_t odd;                // the batch has values that fs_clear took out where some rows see them
    uint32_t wild;               // an output of the piece is no finite number
    uint32_t list[FS_BATCH];
    uint8_t flag[FS_BATCH];
};
template <int D>
struct fs_lds_narrow : fs_list<D, 4> {
    using G = fs_geo<D, true>;
    union {
        struct {                                          // a wave's half tile and its next
            alignas(16) uint8_t q[2 * G::KS * G::QU];
            alignas(16) uint8_t sc[4][G::SETS + 1][1024]; // K scales, V scales
            alignas(16) int32_t cp[4][G::SETS + 1][64];   // and the tile's cells' positions
        };
        alignas(16) float x[4][2][G::NQ * 256];           // at the end: chunks of O on their way
    };
    float ml[4][2][32];
};
template <int D, bool QUANT>
struct fs_lds_wide : fs_list<D, 8> {
    using G = fs_geo<D, QUANT>;
    union {
        alignas(16) uint8_t q4[4][2 * G::KS * G::QU];     // at the start: the four waves' rows
        alignas(16) uint8_t ring[2][2 * G::TB];           // K, V tile; V in units of 8 keys of a dim: [32-key half][16-dim tile][8-key group][dim]
    };
    alignas(16) int32_t cp[2][64];
    alignas(16) uint8_t ql[4][G::QL ? G::QL : 1][1024];   // the Q operands that stay here
};

// x, from which the compiler cannot tell that a value formed of it does not change in a
// loop: hoisted, lane addresses take the registers that the accumulators need.
__device__ __forceinline__ uint32_t fs_opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
// K row i of a half tile is this key: bits 2 and 3 swapped.
__device__ __forceinline__ uint32_t fs_key(uint32_t i) { return (i & 0x13) | (i & 4) << 1 | (i & 8) >> 1; }

// The token of a row (< 2^24), and its head of the group: a reciprocal, right to one, in a tenth of
// the instructions of a division.
__device__ __forceinline__ uint32_t fs_token(const fs_args &a, uint32_t row, uint32_t &g) {
    uint32_t t = (uint32_t)((float)row * a.inv_g);
    int32_t r = (int32_t)(row - t * a.G);
    if (r < 0) --t, r += (int32_t)a.G;
    if (r >= (int32_t)a.G) ++t, r -= (int32_t)a.G;
    g = (uint32_t)r;
    return t;
}

// Nothing moves over it.
#define FS_FENCE() __builtin_amdgcn_sched_barrier(0)

// Value j of the 8 queries of y, as operands have it.
__device__ __forceinline__ _Float16 fs_q(const fs_args &a, const kvm_u32x4 (&y)[2], int j) {
    const uint32_t v = a.q_type == KVM_TYPE_F32 ? y[j >> 2][j & 3] : j & 1 ? y[0][j >> 1] & 0xffff0000u : y[0][j >> 1] << 16;
    return (_Float16)(__uint_as_float(v) * a.q_sign);
}

// Q rows [row_g, row_g + rows) of head h, RG groups of 32: loaded, then as f16 operands into
// LDS (rows past the last: zeros).  8 rows x 8 units of 8 dims an instruction.
template <int D, int RG, int NW>
struct fs_rows {
    static constexpr uint32_t KS = D / 16, QU = 528;
    static constexpr int N = 32 * RG * 2 * KS / (64 * NW);
    kvm_u32x4 y[N][2];
    uint32_t x0;
    __device__ __forceinline__ void load(const fs_args &a, uint32_t h, uint32_t row_g, uint32_t rows) {
        x0 = fs_opaque(threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t x = x0 + 64 * NW * i, b = x >> 6, r = b % (4 * RG) * 8 + (x & 63u) / 8, u = b / (4 * RG) * 8 + (x & 7u);
            uint32_t g;
            const uint32_t t = fs_token(a, row_g + (r < rows ? r : 0u), g);
            const uint64_t e = ((uint64_t)t * a.n_head + h * a.G + g) * D + 8 * u;
            if (a.q_type == KVM_TYPE_F32) __builtin_memcpy(y[i], (const float *)a.q + e, 32);
            else __builtin_memcpy(y[i], (const uint16_t *)a.q + e, 16);
        }
    }
    __device__ __forceinline__ void store(const fs_args &a, uint32_t rows, uint8_t *dst) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t x = x0 + 64 * NW * i, b = x >> 6, r = b % (4 * RG) * 8 + (x & 63u) / 8, u = b / (4 * RG) * 8 + (x & 7u);
            kvm_f16x8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = r < rows ? fs_q(a, y[i], j) : (_Float16)0.0f;
            *(kvm_f16x8 *)(dst + (r >> 5) * (2 * KS * QU) + u * QU + (r & 31u) * 16) = o;
        }
    }
};

// A row's limit: it sees the cells with (unsigned)position below it.
__device__ __forceinline__ uint32_t fs_limit(const fs_args &a, uint32_t row_g, uint32_t rows, uint32_t r) {
    uint32_t g;
    const int32_t qp = r < rows ? a.q_pos[fs_token(a, row_g + r, g)] : -1;
    return qp >= 0 ? (uint32_t)qp + 1u : 0u;
}

// Tile i of a unit's order.
__device__ __forceinline__ uint32_t fs_tile(const fs_seg &sg, uint32_t i) { return i * sg.mult % sg.n_tiles; }      // (n_tiles < 2^16)

// Positions of the cells of tiles b0 + r0 .. in the unit's order: 4 tiles a wave and load.
template <int NW>
struct fs_cells {
    kvm_u32x4 c[4];
    uint32_t x0;
    __device__ __forceinline__ uint32_t at(uint32_t r0, int r) const { return r0 + 4 * NW * r + (x0 >> 4); }
    __device__ __forceinline__ void load(const fs_seg &sg, uint32_t b0, uint32_t r0) {
        x0 = fs_opaque(threadIdx.x);
        uint32_t t = fs_tile(sg, b0 + at(r0, 0));
#pragma unroll
        for (int r = 0; r < 4; ++r) {                     // (past the last: another of the window's)
            c[r] = *(const kvm_u32x4 *)(sg.cell_pos + (uint64_t)t * 64 + 4 * (x0 & 15u));
            t += sg.step;
            t -= t < sg.n_tiles ? 0u : sg.n_tiles;
        }
    }
};

// The tiles b0 .. b0 + nb - 1 in the unit's order that some row sees, in sm.list (bit 31: every
// cell is visible to every row); returns how many.  Every wave takes part; two barriers.
// cells: loaded for r0 = 0.
template <int D, int NW>
__device__ __forceinline__ uint32_t fs_tiles(const fs_seg &sg, fs_list<D, NW> &sm, uint32_t b0, uint32_t nb, uint32_t some_lim,
                                             uint32_t all_lim, fs_cells<NW> &cells) {
    const uint32_t l = fs_opaque(threadIdx.x & 63u), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t r0 = 0;;) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t i = cells.at(r0, r);
            const kvm_u32x4 c = cells.c[r];
            const uint32_t least = min(min(c[0], c[1]), min(c[2], c[3])), most = max(max(c[0], c[1]), max(c[2], c[3]));
            const uint32_t some = (uint32_t)(__builtin_amdgcn_ballot_w64(least < some_lim) >> (l & 48)) & 0xffffu;
            const uint32_t all = (uint32_t)(__builtin_amdgcn_ballot_w64(most < all_lim) >> (l & 48)) & 0xffffu;
            if (i < nb && (l & 15) == 0) sm.flag[i] = (uint8_t)((some != 0) | (all == 0xffffu) << 1);
        }
        r0 += 16 * NW;
        if (r0 >= nb) break;
        cells.load(sg, b0, r0);
    }
    __syncthreads();
    if (threadIdx.x == 0) sm.odd = 0;
    uint32_t n_t = 0;
#pragma unroll
    for (uint32_t x = 0; x < FS_BATCH / 64; ++x) {
        const uint32_t f = 64 * x + l < nb ? sm.flag[64 * x + l] : 0u;
        const uint64_t bal = __builtin_amdgcn_ballot_w64(f & 1u);
        const uint32_t rank = n_t + __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0u));
        if ((f & 1u) && x == w) sm.list[rank] = fs_tile(sg, b0 + 64 * x + l) | (f >> 1) << 31;
        n_t += __popcll(bal);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(n_t);
}

// The scores of a half tile that its cells' positions mask.
__device__ __forceinline__ void fs_mask(kvm_f32x16 &S, const int32_t *cp, uint32_t qlim) {
    asm volatile("" ::: "memory");                        // keep it on the (rare) masked path
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const kvm_u32x4 x = *(const kvm_u32x4 *)(cp + 16 * (i >> 1) + 8 * (fs_opaque(threadIdx.x & 63u) >> 5) + 4 * (i & 1));
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (!(x[r] < qlim)) S[4 * i + r] = -INFINITY;
    }
}

// Values that an f16 operand cannot hold as finite numbers, by these bits of the f16 that is stored:
// infinities and NaN, and of scales also those from 8,192 on, which times -8 are infinite.
template <bool QUANT>
__device__ constexpr uint32_t fs_odd_bits = QUANT ? 0x7000u : 0x7c00u;

// Halves of v (values, or scales of values) whose keys, base .. base + 7, no row sees become
// 0, and so do odd ones where not all rows see the key (0 times them would not be 0): whether there
// are such.
template <bool QUANT>
__device__ __forceinline__ bool fs_clear(kvm_u32x4 &v, uint32_t base, uint64_t seen, uint64_t part) {
    const uint32_t on = (uint32_t)(seen >> base) & 0xffu, pt = (uint32_t)(part >> base) & 0xffu;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t sh = 16 * (i & 1), x = v[i >> 1] >> sh & 0xffffu;
        const bool no = (pt >> i & 1u) && (x & fs_odd_bits<QUANT>) == fs_odd_bits<QUANT>;
        odd |= no;
        if (!(on >> i & 1u) || no) v[i >> 1] &= ~(0xffffu << sh);
    }
    return odd;
}

// p of a row's score with key k of a quantised tile, by the row's two lanes (half a 16-dim step
// each; one step after the other, so that the rare path asks for few registers).
template <int D>
__device__ __forceinline__ float fs_p_again(const fs_args &a, const uint8_t *k_tile, uint32_t k, uint32_t h, uint32_t row, uint32_t g2, float ms) {
    uint32_t g;
    const uint32_t t = fs_token(a, row, g);
    const uint64_t q0 = ((uint64_t)t * a.n_head + h * a.G + g) * D + 8 * g2;
    float s = 0.0f;
#pragma unroll 1
    for (uint32_t d = 0; d < D; d += 16) {
        kvm_u32x4 y[2];
        uint32_t kq[2];
        if (a.q_type == KVM_TYPE_F32) __builtin_memcpy(y, (const float *)a.q + q0 + d, 32);
        else __builtin_memcpy(y, (const uint16_t *)a.q + q0 + d, 16);
        __builtin_memcpy(kq, k_tile + kvm_kq_off(D, k, d + 8 * g2), 8);
        const float sc = kvm_h2f(*(const uint16_t *)(k_tile + kvm_kd_off(D, k, d / 32)));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (float)(int8_t)(kq[j >> 2] >> 8 * (j & 3)) * sc;
            s = fmaf((float)(_Float16)x, (float)fs_q(a, y, j), s);
        }
    }
    return __builtin_amdgcn_exp2f(fmaf(kvm_add_xor32(s), a.c, ms == -INFINITY ? 0.0f : -ms));
}

// What fs_clear took out of keys k0 .. k0 + n_k - 1 of the list's tiles j0, j0 + step, .. is added to the rows
// that see them, in fp32: times the p of the row's score, formed again from the same operands where
// a value is finite (of a large scale).  The wave has `rows` (or 32) rows from row_g on; ms: what O is
// relative to; sx: the wave's own.
template <int D, bool QUANT>
__device__ __forceinline__ void fs_add_odd(kvm_f32x16 (&O)[D / 32], const fs_args &a, const fs_seg &sg, const uint8_t *k_head,
                                           const uint8_t *v_head, const uint32_t *list, uint32_t j0, uint32_t step, uint32_t n_t, uint32_t k0,
                                           uint32_t n_k, uint32_t some_lim, uint32_t all_lim, uint32_t qlim, uint32_t h, uint32_t row_g,
                                           uint32_t rows, float ms, float *sx) {
    const uint32_t l = fs_opaque(threadIdx.x & 63u);
    for (uint32_t j = j0; j < n_t; j += step) {
        const uint32_t e = list[j], t = e & 0x7fffffffu;
        if (e >> 31) continue;
        const uint8_t *v_tile = v_head + (uint64_t)t * fs_geo<D, QUANT>::VB;
        for (uint32_t k = k0; k < k0 + n_k; ++k) {
            const uint32_t cp = (uint32_t)sg.cell_pos[(uint64_t)t * 64 + k];
            if (!(cp < some_lim) || cp < all_lim) continue;
            bool any = false, finite = false;
            for (uint32_t d = l; d < D; d += 64) {
                const uint32_t x = *(const uint16_t *)(QUANT ? v_tile + kvm_vd_off(D, k, d / 32) : v_tile + 2 * kvm_vh_idx(k, d));
                const bool odd = (x & fs_odd_bits<QUANT>) == fs_odd_bits<QUANT>;
                float v = kvm_h2f((uint16_t)x);
                if constexpr (QUANT) v *= (float)((int)(v_tile[kvm_vq_byte(k, d)] >> kvm_vq_shift(k) & 15u) - 8);
                sx[d] = odd ? v : 0.0f;
                any |= odd;
                finite |= odd && v - v == 0.0f;
            }
            if (__builtin_amdgcn_ballot_w64(any) == 0) continue;
            // (at least the smallest number: infinite values under a p that underflows stay infinite;
            // rows past the last: some row's)
            float p = 1.0f;
            if (QUANT && __builtin_amdgcn_ballot_w64(finite) != 0)
                p = fmaxf(fs_p_again<D>(a, k_head + (uint64_t)t * fs_geo<D, true>::KB, k, h, row_g + ((l & 31u) < rows ? l & 31u : 0u), l >> 5, ms),
                          0x1p-126f);
            __builtin_amdgcn_wave_barrier();
            if (cp < qlim) {
#pragma unroll
                for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const kvm_f32x4 v = *(const kvm_f32x4 *)(sx + 32 * dt + 8 * x + 4 * (l >> 5));
#pragma unroll
                        for (int r = 0; r < 4; ++r) O[dt][4 * x + r] = fmaf(v[r], p, O[dt][4 * x + r]);
                    }
                    FS_FENCE();
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Whether a lane of the workgroup has a z that is no number.  (The flag is cleared at the start of the
// first time through a piece only: whoever is first to begin again writes none that others still read.)
template <int D, int NW>
__device__ __forceinline__ bool fs_wild(fs_list<D, NW> &sm, float z) {
    if (z != z) sm.wild = 1;
    KVM_LDS_BARRIER();
    return __builtin_amdgcn_readfirstlane(sm.wild) != 0;
}

// Direct copies to LDS (lane l writes 16 or 4 bytes at M0 + 16 l or 4 l), issued from asm, so
// that the compiler adds no wait for them; the asm restores M0, which the compiler reserves.
// Whoever reads waits by vmcnt first.
__device__ __forceinline__ void fs_copy16(const uint8_t *src, uint32_t off, void *dst) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(off), "s"((uint32_t)(uintptr_t)(fs_lds_ptr)dst), "s"(src) : "memory");
}
__device__ __forceinline__ void fs_copy16(const uint8_t *lane_src, void *dst) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(lane_src), "s"((uint32_t)(uintptr_t)(fs_lds_ptr)dst) : "memory");
}
__device__ __forceinline__ void fs_copy4(const int32_t *src, uint32_t off, void *dst) {
    uint32_t m0_saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0_saved) : "v"(off), "s"((uint32_t)(uintptr_t)(fs_lds_ptr)dst), "s"(src) : "memory");
}

// A piece of a narrow unit (32 rows over a quantised window): tiles [i_lo, i_hi) in the
// unit's order.  A tile of 256 dims is ~1,650 instructions of a wave, 930 of them its conversion,
// and 64 MFMAs (2,048 cycles): the issue of two waves a SIMD bounds it (~2.1 us a tile and
// workgroup), next to the memory where no two units read the same tiles (all in the L2: 55 of 66
// us), and for short pieces the start (5.6 us to the first half tile) and the sums' meeting
// (2.2).  8 lanes x 6 rows of 4 heads over 32,768 + 2,048 cells of q8_0: 30 us for 74.5 MB, 2.5
// TB/s; 16 x 18 over 5,003 + 8,192 of q4_0: 64 us, 154 MB.  (256 dims take all 256 registers and one
// more, spilled before the loop and read back after it.)
// True: an output is no finite number, and the piece is to be formed again with CAREFUL.
template <int D, bool CAREFUL>
__device__ __forceinline__ bool fs_narrow(const fs_args &a, const fs_seg &sg, fs_lds_narrow<D> &sm, uint32_t rt, uint32_t h, uint32_t slot,
                                          uint32_t i_lo, uint32_t i_hi) {
    using G = fs_geo<D, true>;
    constexpr int KS = G::KS, NB = G::NB, DT = G::DT, NQ = G::NQ, SETS = G::SETS;
    constexpr uint32_t KB = G::KB, VB = G::VB, QU = G::QU;
    const uint32_t l = fs_opaque(threadIdx.x & 63u), g2 = l >> 5, m2 = l & 31u;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rows = min(32u, sg.n_rows - 32 * rt), row_g = sg.row0 + 32 * rt;

    if (!CAREFUL && threadIdx.x == 0) sm.wild = 0;
    // the loads of the start, all issued before any is used
    fs_cells<4> cells;
    cells.load(sg, i_lo, 0);
    const uint32_t qlim = fs_limit(a, row_g, rows, m2);
    {
        fs_rows<D, 1, 4> q;
        q.load(a, h, row_g, rows);
        q.store(a, rows, sm.q);
    }
    const uint32_t all_lim = CAREFUL ? 0u : kvm_wave_min_u32(m2 < rows ? qlim : 0xffffffffu), some_lim = ~kvm_wave_min_u32(~qlim);

    kvm_f32x16 O[DT];
    float ms = -INFINITY, lp = 0.0f;     // the row's reference maximum (times c), the lane's share of its sum
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] = 0.0f;

    // operand addresses of a lane
    const uint32_t key = fs_key(m2);
    const uint32_t k_lane = ((key >> 4) * (NB / 2) * 64 + 16 * g2 + (key & 15)) * 16, v_lane = ((m2 >> 4) * 64 + 16 * g2 + (m2 & 15)) * 8;
    const uint8_t *const k_head = sg.k + (uint64_t)h * sg.n_tiles * KB, *const v_head = sg.v + (uint64_t)h * sg.n_tiles * VB;

    for (uint32_t b0 = i_lo; b0 < i_hi; b0 += FS_BATCH) {
        if (b0 != i_lo) cells.load(sg, b0, 0);
        const uint32_t n_t = fs_tiles<D, 4>(sg, sm, b0, min(FS_BATCH, i_hi - b0), some_lim, all_lim, cells);      // (its barriers: Q, too)

        // The wave's half tiles: half w & 1 of list entries w / 2, w / 2 + 2, ..  Their
        // registers are loaded for the next one where this one's are used up; past the wave's
        // last the bounds let nothing through.
        const uint32_t half = w & 1;
        kvm_u32x4 kr[SETS][NB];
        uint32_t vq[SETS][2 * DT];
        auto rsrc = [&](const uint8_t *head, uint32_t e, uint32_t bytes, bool more) {
            return __builtin_amdgcn_make_buffer_rsrc((void *)(head + (uint64_t)(e & 0x7fffffffu) * bytes), (short)0, more ? bytes : 0u, 0x00020000);
        };
        auto load_k = [&](__amdgpu_buffer_rsrc_t r, int set, int i) {
            kr[set][i] = __builtin_amdgcn_raw_buffer_load_b128(r, k_lane + (i & 1) * 512, half * NB * 1024 + (i >> 1) * 1024, 0);
        };
        auto load_v = [&](__amdgpu_buffer_rsrc_t r, int set, int i) {
            vq[set][i] = __builtin_amdgcn_raw_buffer_load_b32(r, v_lane + (i & 1) * 256, half * 4 + (i >> 1) * 1024, 0);
        };
        // lanes below 4 NB: the half's K scales, 32 .. 32 + 4 NB - 1: its V scales (units of 8 keys of a
        // block); of 128 dims the other lanes copy the same again, which nobody reads
        auto copies = [&](uint32_t e, uint32_t buf) {
            const uint32_t t = e & 0x7fffffffu, ln = fs_opaque(l), x = ln & (4u * NB - 1);
            const uint8_t *const src = ln < 32 ? k_head + (uint64_t)t * KB + 64 * D + half * (64u * NB) + 16 * x
                                               : v_head + (uint64_t)t * VB + 32 * D + (x >> 2) * 128 + half * 64 + (x & 3u) * 16;
            fs_copy16(src, sm.sc[w][buf]);
            fs_copy4(sg.cell_pos + (uint64_t)t * 64, 4u * ln, &sm.cp[w][buf][0]);
        };
        auto entry = [&](uint32_t j) { return __builtin_amdgcn_readfirstlane(sm.list[min(j, n_t - 1)]); };
        const uint32_t j0 = w >> 1;
        if (j0 < n_t) {
#pragma unroll
            for (int x = 0; x < SETS; ++x) {
                const uint32_t e = entry(j0 + 2 * x);
                const bool more = j0 + 2 * x < n_t;
                copies(e, x);
#pragma unroll
                for (int i = 0; i < NB; ++i) load_k(rsrc(k_head, e, KB, more), x, i);
#pragma unroll
                for (int i = 0; i < 2 * DT; ++i) load_v(rsrc(v_head, e, VB, more), x, i);
            }
        }
        uint32_t buf = 0;
        auto item = [&](uint32_t j, auto which) {
            constexpr int set = decltype(which)::value;
            // the half tile's copies: its registers' loads, and the next ones', are younger
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"(SETS * (NB + 2 * DT) + 2 * (SETS - 1)) : "memory");
            const uint32_t e = entry(j), en = entry(j + 2 * SETS);
            const bool more = j + 2 * SETS < n_t, full = e >> 31;
            const auto rk = rsrc(k_head, en, KB, more), rv = rsrc(v_head, en, VB, more);
            if (!full) {
                asm volatile("" ::: "memory");            // keep it on this (rare) path
                const uint32_t lo = fs_opaque(l), cp = (uint32_t)sm.cp[w][buf][lo];
                const uint64_t seen = __builtin_amdgcn_ballot_w64(cp < some_lim), part = seen & ~__builtin_amdgcn_ballot_w64(cp < all_lim);
                // lane l has the scales of 8 keys of a block
                if (lo < 4u * NB) {
                    kvm_u32x4 *const at = (kvm_u32x4 *)(sm.sc[w][buf] + 512 + 16 * lo);
                    kvm_u32x4 scv = *at;
                    if (fs_clear<true>(scv, 32 * half + 8 * (lo & 3u), seen, part)) sm.odd = 1;
                    *at = scv;
                }
            }
            copies(en, buf ? buf - 1 : SETS);

            // ---- S^T of 32 keys: K operand i + 1 is made while the MFMA of i runs; what
            // comes from LDS is read two steps ahead
            kvm_f32x16 S;
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = 0.0f;
            uint32_t ksc[NB];                         // the scales of the lane's key
            {
                const uint32_t k = fs_key(fs_opaque(l) & 31u);
#pragma unroll
                for (int b = 0; b < NB; ++b) ksc[b] = *(const uint16_t *)(sm.sc[w][buf] + ((k >> 4) * NB + b) * 32 + 2 * (k & 15));
            }
            const uint32_t lq = fs_opaque(l);
            const uint8_t *const sq = sm.q + (lq >> 5) * QU + (lq & 31u) * 16;
            // operands in the order of the K loads: (block pair, 16-dim half | block of the pair)
            auto k_op = [&](int i) {
                const kvm_u32x4 x = kr[set][i >> 1];
                return pf_q8(x[2 * (i & 1)], x[2 * (i & 1) + 1], ksc[2 * (i >> 2) + (i & 1)]);
            };
            auto q_op = [&](int i) { return *(const kvm_f16x8 *)(sq + 2 * (4 * (i >> 2) + 2 * (i & 1) + (i >> 1 & 1)) * QU); };
            kvm_f16x8 kop = k_op(0), qr[3] = {q_op(0), q_op(1)};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                if (i + 2 < KS) qr[(i + 2) % 3] = q_op(i + 2);
                FS_FENCE();
                S = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, qr[i % 3], S, 0, 0, 0);
                if (i + 1 < KS) kop = k_op(i + 1);
                if (i & 1) load_k(rk, set, i >> 1);
                FS_FENCE();
            }

            // ---- softmax: P as f16 operands
            if (!full) fs_mask(S, &sm.cp[w][buf][32 * half], qlim);
            float x = S[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) x = fmaxf(x, S[r]);
            x = kvm_max_xor32(x);
            const bool up = fmaf(x, a.c, -ms) > FS_LAZY;      // false for a row with nothing visible yet
            if (__builtin_amdgcn_ballot_w64(up) != 0) {
                const float mnew = up ? x * a.c : ms;
                const float alpha = up ? __builtin_amdgcn_exp2f(ms - mnew) : 1.0f;
                ms = mnew;
                lp *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) O[dt] *= alpha;
            }
            const float ref = ms == -INFINITY ? 0.0f : ms;
            kvm_f16x8 pb[2];
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                // the row sum takes p before its rounding to the f16 operand: within
                // 2^-11 of it per element
                const float y = __builtin_amdgcn_exp2f(fmaf(S[r], a.c, -ref));
                pb[r >> 3][r & 7] = (_Float16)y;
                sum += y;
            }
            lp += sum;

            // ---- O^T += V^T P^T
            kvm_u32x4 vs[3];
            const uint8_t *const sv = sm.sc[w][buf] + 512 + (fs_opaque(l) >> 5) * 16;
            auto v_scale = [&](int i) { vs[i % 3] = *(const kvm_u32x4 *)(sv + ((i >> 1) * 4 + 2 * (i & 1)) * 16); };
            v_scale(0);
            v_scale(1);
            kvm_f16x8 vop = pf_q4(vq[set][0], vs[0]);
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                if (i + 2 < 2 * DT) v_scale(i + 2);
                FS_FENCE();
                O[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop, pb[i & 1], O[i >> 1], 0, 0, 0);
                if (i + 1 < 2 * DT) vop = pf_q4(vq[set][i + 1], vs[(i + 1) % 3]);
                load_v(rv, set, i);
                FS_FENCE();
            }
            buf = buf == SETS ? 0 : buf + 1;
        };
        for (uint32_t j = j0; j < n_t; j += 2) {
            item(j, std::integral_constant<int, 0>{});
            if constexpr (SETS == 2) {
                if ((j += 2) >= n_t) break;
                item(j, std::integral_constant<int, 1>{});
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last items' copies, which nobody reads)
        if (__builtin_amdgcn_readfirstlane(sm.odd))
            fs_add_odd<D, true>(O, a, sg, k_head, v_head, sm.list, j0, 2, n_t, 32 * half, 32, some_lim, all_lim, qlim, h, row_g, rows, ms,
                                sm.odd_v[w]);
    }

    // ---- the waves' sums: one maximum, then each wave's quarter of the dims from the others,
    // two waves' and the third's
    const float lr = kvm_add_xor32(lp);
    if (lr != lr) ms = 0.0f;                              // (scores that are no numbers have no maximum; the sums are not empty)
    if (g2 == 0) {
        sm.ml[w][0][m2] = ms;
        sm.ml[w][1][m2] = lr;
    }
    __syncthreads();
    float M = sm.ml[0][0][m2], L = 0.0f;
#pragma unroll
    for (int x = 1; x < 4; ++x) M = fmaxf(M, sm.ml[x][0][m2]);
    const float top = M == -INFINITY ? 0.0f : M;          // (a wave that saw nothing of the row: weight, sum and O are 0)
#pragma unroll
    for (int x = 0; x < 4; ++x) L += sm.ml[x][1][m2] * __builtin_amdgcn_exp2f(sm.ml[x][0][m2] - top);
    const float wgt = __builtin_amdgcn_exp2f(ms - top);
    // quad i of O: dims 8 i + 4 g2 .. + 3 of the lane's row, weighted
    auto quad = [&](int i) {
        kvm_f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = O[i >> 2][4 * (i & 3) + k] * wgt;
        return v;
    };
    kvm_f32x4 acc[NQ];
    for (int round = 0; round < 2; ++round) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int k = (q - w) & 3;                    // the (k - 1)-th of the waves that give to q
            if (k == 0) {
                if (round == 0) {
#pragma unroll
                    for (int x = 0; x < NQ; ++x) acc[x] = quad(q * NQ + x);
                }
            } else if ((k - 1) >> 1 == round) {
#pragma unroll
                for (int x = 0; x < NQ; ++x) *(kvm_f32x4 *)(sm.x[q][(k - 1) & 1] + 256 * x + 4 * l) = quad(q * NQ + x);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (round == 1 && k == 1) break;
#pragma unroll
            for (int x = 0; x < NQ; ++x) acc[x] += *(const kvm_f32x4 *)(sm.x[w][k] + 256 * x + 4 * l);
        }
        if (round == 0) __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) *(kvm_f32x4 *)(a.ws_o + ((uint64_t)slot * (D / 8) + w * NQ + x) * 256 + 4 * l) = acc[x];
    if (w == 0 && g2 == 0) {
        float *ml = a.ws_ml + ((uint64_t)slot * 32 + m2) * 2;
        ml[0] = M;
        ml[1] = L;
    }
    if (CAREFUL) return false;
    float z = 0.0f;
#pragma unroll
    for (int x = 0; x < 4 * NQ; ++x) z = fmaf(acc[x >> 2][x & 3], 0.0f, z);
    return fs_wild(sm, z);
}

// x stays where it is: nothing moves over it, the MFMA that wrote it included.
#define FS_PIN(x)                                    \
    do {                                             \
        asm volatile("" : "+v"(x) : : "memory");     \
        FS_FENCE();                                  \
    } while (0)

// A piece of a wide unit.  A tile of 256 dims is 64 MFMAs of an attention wave (2,048 cycles) in
// ~4,600: its softmax and the other wave's conversion share the SIMD's issue, at the clock that
// the power limit leaves.  768 rows of 4 heads over 32,768 cells of q8_0 (103 GFLOP): 137 us, 750
// TFLOP/s.  36 tokens x 4 rows of 8 heads of 128 dims over 8,192 + 12 x 1,024 f16 cells: 24 us for
// 84 MB, the prefix read twice (without the attention waves' work 17, without the copies 25).
template <int D, bool QUANT, bool CAREFUL>
__device__ __forceinline__ bool fs_wide_piece(const fs_args &a, const fs_seg &sg, fs_lds_wide<D, QUANT> &sm, uint32_t rt, uint32_t h,
                                              uint32_t slot, uint32_t i_lo, uint32_t i_hi) {
    using G = fs_geo<D, QUANT>;
    constexpr int KS = G::KS, NB = G::NB, DT = G::DT;     // (2 DT = KS)
    constexpr uint32_t KB = G::KB, VB = G::VB, TB = G::TB, QU = G::QU;
    const uint32_t l = fs_opaque(threadIdx.x & 63u);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = w & 3;
    const uint32_t rows = min(128u, sg.n_rows - 128 * rt), row_g = sg.row0 + 128 * rt;

    if (!CAREFUL && threadIdx.x == 0) sm.wild = 0;
    // the loads of the start, all issued before any is used
    fs_cells<8> cells;
    cells.load(sg, i_lo, 0);
    const uint32_t lim0 = fs_limit(a, row_g, rows, l), lim1 = fs_limit(a, row_g, rows, l + 64);
    {
        fs_rows<D, 4, 8> q;
        q.load(a, h, row_g, rows);
        q.store(a, rows, sm.q4[0]);
    }
    const uint32_t all_lim = CAREFUL ? 0u : kvm_wave_min_u32(min(l < rows ? lim0 : 0xffffffffu, l + 64 < rows ? lim1 : 0xffffffffu));
    const uint32_t some_lim = ~kvm_wave_min_u32(~max(lim0, lim1));
    const uint8_t *const k_head = sg.k + (uint64_t)h * sg.n_tiles * KB, *const v_head = sg.v + (uint64_t)h * sg.n_tiles * VB;
    uint32_t n_t = fs_tiles<D, 8>(sg, sm, i_lo, min(FS_BATCH, i_hi - i_lo), some_lim, all_lim, cells);   // (its barriers: Q, too)

    float z = 0.0f;
    // Both roles take the same barriers: one when Q is in registers, and for a batch of tiles
    // one when the first is in LDS, one a tile, and those of the next batch's list.
    if (w < 4) {
        // ======== 32 rows: S^T = K Q^T, softmax, O^T += V^T P^T
        const float c = a.c;
        const uint32_t lc = fs_opaque(l), m2 = lc & 31u, g2 = lc >> 5;
        // operand rings: R1 where a softmax is under way (registers), R0 elsewhere
        constexpr std::integral_constant<int, D == 256 ? 4 : 6> R0;
        constexpr std::integral_constant<int, D == 256 ? 2 : 4> R1;
        kvm_f32x16 O[DT];
        float ms = -INFINITY, lp = 0.0f;
        kvm_f16x8 qop[KS];       // lane (g2, m2): Q[row m2][16 ks + 8 g2 .. + 7]
        auto in_lds = [](int ks) { return G::QL && ks % 3 == 1; };
        uint8_t *const ql = sm.ql[rg][0] + 16 * lc;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const kvm_f16x8 v = *(const kvm_f16x8 *)(sm.q4[rg] + (2 * ks + g2) * QU + m2 * 16);
            if (in_lds(ks)) *(kvm_f16x8 *)(ql + ks / 3 * 1024) = v;
            else qop[ks] = v;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[dt][r] = 0.0f;
        const uint32_t qlim = fs_limit(a, row_g, rows, 32 * rg + m2);
        const uint32_t key = fs_key(m2);
        const uint32_t k_ofs = ((key >> 4) * NB * 64 + 16 * g2 + (key & 15)) * 16, v_ofs = ((m2 >> 4) * 64 + 16 * g2 + (m2 & 15)) * 16;
        const bool active = 32u * rg < rows;              // not a wave of padding rows
        KVM_LDS_BARRIER();                                // Q is in registers

        // S^T of a half tile: K operand ks at sk + .., KR - 1 ahead; between(ks) follows MFMA ks
        auto scores = [&](auto ring, const uint8_t *sk, auto &&between) {
            constexpr int KR = decltype(ring)::value;
            kvm_f32x16 S;
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = 0.0f;
            kvm_f16x8 kr[KR];
            auto ld = [&](int ks) { return *(const kvm_f16x8 *)(sk + ks * 512); };
            kvm_f16x8 qn;
            auto ldq = [&](int ks) {
                if (in_lds(ks)) qn = *(const kvm_f16x8 *)(sm.ql[rg][0] + 16 * fs_opaque(l) + ks / 3 * 1024);
            };
            ldq(1);
#pragma unroll
            for (int i = 0; i < KR - 1; ++i) kr[i] = ld(i);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + KR - 1 < KS) kr[(ks + KR - 1) % KR] = ld(ks + KR - 1);
                FS_FENCE();
                S = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[ks % KR], in_lds(ks) ? qn : qop[ks], S, 0, 0, 0);
                if (in_lds(ks) && ks + 3 < KS) ldq(ks + 3);
                between(ks);
                FS_PIN(S);
            }
            return S;
        };
        // O^T += V^T P^T: operand i = (16 keys i / DT, dim tile i % DT)
        auto accumulate = [&](auto ring, const uint8_t *sv, const kvm_f16x8 (&pb)[2], auto &&between) {
            constexpr int VR = decltype(ring)::value;
            kvm_f16x8 vr[VR];
            auto ld = [&](int i) { return *(const kvm_f16x8 *)(sv + (i % DT) * 2048 + (i / DT) * 512); };
#pragma unroll
            for (int i = 0; i < VR - 1; ++i) vr[i] = ld(i);
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                if (i + VR - 1 < 2 * DT) vr[(i + VR - 1) % VR] = ld(i + VR - 1);
                FS_FENCE();
                O[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vr[i % VR], pb[i / DT], O[i % DT], 0, 0, 0);
                between(i);
                FS_PIN(O[i % DT]);
            }
        };
        // The softmax of a half tile in KS steps, taken between another's MFMAs: the maximum
        // (KS / 4 steps), the running maximum's move (one), the probabilities (KS / 2).
        float x = 0.0f, ref = 0.0f, alpha = 1.0f, sum = 0.0f;
        bool moved = false;
        auto soft = [&](const kvm_f32x16 &S, kvm_f16x8 (&pb)[2], int i) {
            constexpr int NM = KS / 4, EM = 16 / NM, EP = 16 / (KS / 2);
            if (i < NM) {
#pragma unroll
                for (int r = 0; r < EM; ++r) x = i == 0 && r == 0 ? S[0] : fmaxf(x, S[EM * i + r]);
            } else if (i == NM) {
                x = kvm_max_xor32(x);
                const bool up = fmaf(x, c, -ms) > FS_LAZY;        // false for a row with nothing visible yet
                moved = __builtin_amdgcn_ballot_w64(up) != 0;
                const float mnew = up ? x * c : ms;
                alpha = up ? __builtin_amdgcn_exp2f(ms - mnew) : 1.0f;
                ms = mnew;
                ref = ms == -INFINITY ? 0.0f : ms;
                sum = 0.0f;
            } else if (i >= KS / 2) {
#pragma unroll
                for (int j = 0; j < EP; j += 2) {
                    // (the row sum takes p before its rounding)
                    const int r = EP * (i - KS / 2) + j;
                    const float y0 = __builtin_amdgcn_exp2f(fmaf(S[r], c, -ref)), y1 = __builtin_amdgcn_exp2f(fmaf(S[r + 1], c, -ref));
                    kvm_f16x2 h = {(_Float16)y0, (_Float16)y1};
                    sum += y0;
                    sum += y1;
                    asm volatile("" : "+v"(h), "+v"(sum)); // here, not where they are used
                    pb[r >> 3][r & 7] = h[0];
                    pb[r >> 3][(r & 7) + 1] = h[1];
                }
            }
        };
        // what the moved maximum asks of the sums so far
        auto settle = [&]() {
            if (moved) {
                asm volatile("" ::: "memory");            // keep it on this (rare) path
                lp *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) O[dt] *= alpha;
            }
            lp += sum;
        };
        auto nothing = [](int) {};

        for (uint32_t b0 = i_lo;;) {
            KVM_LDS_BARRIER();                            // the first tile is in LDS
            for (uint32_t k = 0; k < n_t; ++k) {
                if (!active) {
                    KVM_LDS_BARRIER();
                    continue;
                }
                const bool masked = (__builtin_amdgcn_readfirstlane(sm.list[k]) >> 31) == 0;
                const uint8_t *sk = sm.ring[k & 1u] + k_ofs, *sv = sm.ring[k & 1u] + TB + v_ofs;
                kvm_f16x8 pb[2], pb1[2];
                kvm_f32x16 S0 = scores(R0, sk, nothing);
                if (masked) fs_mask(S0, &sm.cp[k & 1u][0], qlim);
                kvm_f32x16 S1 = scores(R1, sk + 2 * NB * 1024, [&](int i) { soft(S0, pb, i); });
                settle();
                if (masked) fs_mask(S1, &sm.cp[k & 1u][32], qlim);
                accumulate(R1, sv, pb, [&](int i) { soft(S1, pb1, i); });
                settle();
                accumulate(R0, sv + TB / 2, pb1, nothing);
                KVM_LDS_BARRIER();
            }
            if (active && __builtin_amdgcn_readfirstlane(sm.odd))
                fs_add_odd<D, QUANT>(O, a, sg, k_head, v_head, sm.list, 0, 1, n_t, 0, 64, some_lim, all_lim, qlim, h, row_g + 32 * rg,
                                     rows - 32 * rg, ms, sm.odd_v[w]);
            b0 += FS_BATCH;
            if (b0 >= i_hi) break;
            fs_cells<8> next;
            next.load(sg, b0, 0);
            n_t = fs_tiles<D, 8>(sg, sm, b0, min(FS_BATCH, i_hi - b0), some_lim, all_lim, next);
        }
        if (active) {
            // quad i of O: dims 8 i + 4 g2 .. + 3 of the lane's row
            const float lr = kvm_add_xor32(lp);
            if (lr != lr) ms = 0.0f;                      // (scores that are no numbers have no maximum; the sums are not empty)
            const uint32_t le = fs_opaque(l);
            float *o = a.ws_o + (uint64_t)(slot + rg) * 32 * D + 4 * le;
            if (__builtin_amdgcn_ballot_w64(ms != -INFINITY) != 0) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *(kvm_f32x4 *)(o + 256 * i) = kvm_f32x4{O[i >> 2][4 * (i & 3)], O[i >> 2][4 * (i & 3) + 1], O[i >> 2][4 * (i & 3) + 2], O[i >> 2][4 * (i & 3) + 3]};
            }
            if (le < 32) {
                float *ml = a.ws_ml + ((uint64_t)(slot + rg) * 32 + le) * 2;
                ml[0] = ms;
                ml[1] = lr;
            }
            float zs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) zs[r & 3] = fmaf(O[dt][r], 0.0f, zs[r & 3]);
            z = (zs[0] + zs[1]) + (zs[2] + zs[3]);
        }
    } else {
        // ======== tile k + 1 into one buffer while the others work on tile k
        const int pw = w - 4;
        KVM_LDS_BARRIER();                                // Q is in registers
        auto tile = [&](uint32_t k) { return __builtin_amdgcn_readfirstlane(sm.list[k < n_t ? k : n_t - 1]); };
        auto cells_of = [&](uint32_t e) { return sg.cell_pos[(uint64_t)(e & 0x7fffffffu) * 64 + l]; };
        // what the tile's masks say: the keys that some row sees, and those that not all do
        auto masks = [&](int32_t cp, uint64_t &seen, uint64_t &part) {
            seen = __builtin_amdgcn_ballot_w64((uint32_t)cp < some_lim);
            part = seen & ~__builtin_amdgcn_ballot_w64((uint32_t)cp < all_lim);
        };
        for (uint32_t b0 = i_lo;;) {
            if constexpr (QUANT) {
                // The quantised tile goes through registers (two sets: tiles k + 2 and k + 3 are
                // in flight while tile k + 1 is converted).  Thread (pw, l): K units 4 j + pw
                // (lane l of (sub, block pair)), V dim tiles VJ pw + j.
                constexpr int KJ = D / 64, VJ = D / 64, VB2 = VJ / 2;
                struct raw_tile {
                    kvm_u32x4 k[KJ];
                    uint32_t kd[KJ][2];
                    kvm_u32x2 v[VJ];
                    kvm_u32x4 vs[VB2][2];
                    int32_t cp;
                    uint32_t e;
                };
                raw_tile rt2[2] = {};
                auto load = [&](raw_tile &r, uint32_t e) {
                    const uint32_t ln = fs_opaque(l), t = e & 0x7fffffffu;
                    const uint8_t *kt = k_head + (uint64_t)t * KB, *vt = v_head + (uint64_t)t * VB;
#pragma unroll
                    for (int j = 0; j < KJ; ++j) {
                        const uint32_t sp = 4 * j + pw, s = sp / (NB / 2), pr = sp % (NB / 2);
                        r.k[j] = *(const kvm_u32x4 *)(kt + (sp * 64 + ln) * 16);
                        r.kd[j][0] = *(const uint16_t *)(kt + kvm_kd_off(D, 16 * s + (ln & 15), 2 * pr));
                        r.kd[j][1] = *(const uint16_t *)(kt + kvm_kd_off(D, 16 * s + (ln & 15), 2 * pr + 1));
                    }
#pragma unroll
                    for (int j = 0; j < VJ; ++j) r.v[j] = *(const kvm_u32x2 *)(vt + ((VJ * pw + j) * 64 + ln) * 8);
#pragma unroll
                    for (int b = 0; b < VB2; ++b)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) r.vs[b][ks] = *(const kvm_u32x4 *)(vt + 32 * D + (((VB2 * pw + b) * 2 + ks) * 4 + (ln >> 4)) * 16);
                    r.cp = cells_of(e);
                    r.e = e;
                };
                auto convert = [&](raw_tile &r, uint32_t buf) {
                    if (!(r.e >> 31)) {
                        asm volatile("" ::: "memory");    // keep it on this (rare) path
                        uint64_t seen, part;
                        masks(r.cp, seen, part);
                        bool odd = false;
#pragma unroll
                        for (int b = 0; b < VB2; ++b)
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks) odd |= fs_clear<true>(r.vs[b][ks], 32 * ks + 8 * (fs_opaque(l) >> 4), seen, part);
                        if (odd) sm.odd = 1;
                    }
                    uint8_t *dk = sm.ring[buf] + 16 * fs_opaque(l), *dv = dk + TB;
#pragma unroll
                    for (int j = 0; j < KJ; ++j) {
                        const uint32_t sp = 4 * j + pw, s = sp / (NB / 2), pr = sp % (NB / 2);
#pragma unroll
                        for (int i = 0; i < 2; ++i) *(kvm_f16x8 *)(dk + (s * NB + 2 * pr + i) * 1024) = pf_q8(r.k[j][2 * i], r.k[j][2 * i + 1], r.kd[j][i]);
                    }
#pragma unroll
                    for (int j = 0; j < VJ; ++j)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) *(kvm_f16x8 *)(dv + ks * (TB / 2) + (VJ * pw + j) * 1024) = pf_q4(r.v[j][ks], r.vs[j / 2][ks]);
                    if (pw == 0) sm.cp[buf][l] = r.cp;
                };
                if (n_t != 0) {
                    load(rt2[0], tile(0));
                    load(rt2[1], tile(1));
                    convert(rt2[0], 0);
                }
                KVM_LDS_BARRIER();                        // the first tile is in LDS
                if (2 < n_t) load(rt2[0], tile(2));
                auto step = [&](raw_tile &r, uint32_t k) {
                    if (k + 1 < n_t) convert(r, (k + 1) & 1u);
                    if (k + 3 < n_t) load(r, tile(k + 3));
                    KVM_LDS_BARRIER();
                };
                uint32_t k = 0;
                for (; k + 2 <= n_t; k += 2) {
                    step(rt2[1], k);
                    step(rt2[0], k + 1);
                }
                if (k < n_t) step(rt2[1], k);
            } else {
                // An f16 window's tiles are copied.  Its V tile holds the two key halves of a
                // dim side by side, so the copies read every second unit of a dim tile.
                constexpr int NC = (int)TB / 4096;        // 1 KB copies of a wave, of K and of V
                auto bring = [&](uint32_t e, uint32_t buf) {
                    const uint32_t t = e & 0x7fffffffu;
                    uint8_t *const dst = sm.ring[buf];
                    const uint8_t *kt = k_head + (uint64_t)t * TB, *vt = v_head + (uint64_t)t * TB;
                    const int32_t cp = cells_of(e);
#pragma unroll
                    for (int i = 0; i < NC; ++i) fs_copy16(kt + (pw * NC + i) * 1024u, 16u * fs_opaque(l), dst + (pw * NC + i) * 1024u);
#pragma unroll
                    for (int i = 0; i < NC; ++i) {
                        const uint32_t x = pw * NC + i;   // key half, dim tile
                        fs_copy16(vt + (x % (D / 16)) * 2048u + (x / (D / 16)) * 16u, 32u * fs_opaque(l), dst + TB + x * 1024u);
                    }
                    if (pw == 0) sm.cp[buf][l] = cp;
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    if (!(e >> 31)) {
                        asm volatile("" ::: "memory");
                        uint64_t seen, part;
                        masks(cp, seen, part);
                        const uint32_t ln = fs_opaque(l);
                        bool odd = false;
                        for (int i = 0; i < NC; ++i) {
                            const uint32_t x = pw * NC + i;
                            kvm_u32x4 *const u = (kvm_u32x4 *)(dst + TB + x * 1024u + 16 * ln);
                            kvm_u32x4 v = *u;
                            odd |= fs_clear<false>(v, 32 * (x / (D / 16)) + 8 * (ln >> 4), seen, part);
                            *u = v;
                        }
                        if (odd) sm.odd = 1;
                    }
                };
                if (n_t != 0) bring(tile(0), 0);
                KVM_LDS_BARRIER();                        // the first tile is in LDS
                for (uint32_t k = 0; k < n_t; ++k) {
                    if (k + 1 < n_t) bring(tile(k + 1), (k + 1) & 1u);
                    KVM_LDS_BARRIER();
                }
            }
            b0 += FS_BATCH;
            if (b0 >= i_hi) break;
            fs_cells<8> next;
            next.load(sg, b0, 0);
            n_t = fs_tiles<D, 8>(sg, sm, b0, min(FS_BATCH, i_hi - b0), some_lim, all_lim, next);
        }
    }
    return !CAREFUL && fs_wild(sm, z);
}

// The second (rare) time through a piece starts from what the compiler takes for other values: formed
// from the same ones, what both need is kept from the first and takes its registers.
#define FS_AGAIN(rt, h, slot, i_lo, i_hi) asm volatile("" : "+s"(rt), "+s"(h), "+s"(slot), "+s"(i_lo), "+s"(i_hi) : : "memory")

// The workgroup's piece.
template <bool WIDE, class F>
__device__ __forceinline__ void fs_piece(const fs_args &a, F &&piece) {
    // (loads that wait for no other)
    const uint32_t piece0 = a.piece0[threadIdx.x & 63u], last0 = a.piece0[64], n_before = a.wide, n = WIDE ? n_before : a.narrow;
    // neighbours on one XCD
    const uint32_t each = (n + 7) / 8;
    uint32_t p = n < 8 ? blockIdx.x : (blockIdx.x & 7u) * each + (blockIdx.x >> 3);
    if (p >= n) return;
    if (!WIDE) p += n_before;
    const uint32_t s = __builtin_amdgcn_readfirstlane(last0 <= p ? 64u : (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(piece0 <= p)) - 1);
    const fs_seg &sg = a.seg[s];
    const uint32_t n_rt = fs_row_tiles(WIDE, sg.n_rows), x = p - a.piece0[s], y = x / n_rt, h = y / sg.pieces, j = y - h * sg.pieces;
    const uint32_t i_lo = j * sg.per + min(j, sg.more);
    piece(sg, x - y * n_rt, h, WIDE ? 4 * p : 4 * n_before + (p - n_before), i_lo, i_lo + sg.per + (j < sg.more ? 1u : 0u));
}

template <int D, bool QUANT>
__global__ void __launch_bounds__(512) k_fs_wide(fs_args a) {
    __shared__ fs_lds_wide<D, QUANT> sm;
    fs_piece<true>(a, [&](const fs_seg &sg, uint32_t rt, uint32_t h, uint32_t slot, uint32_t i_lo, uint32_t i_hi) {
        if (fs_wide_piece<D, QUANT, false>(a, sg, sm, rt, h, slot, i_lo, i_hi)) {
            FS_AGAIN(rt, h, slot, i_lo, i_hi);
            fs_wide_piece<D, QUANT, true>(a, sg, sm, rt, h, slot, i_lo, i_hi);
        }
    });
}

template <int D>
__global__ void __launch_bounds__(256, 2) k_fs_narrow(fs_args a) {
    __shared__ fs_lds_narrow<D> sm;
    fs_piece<false>(a, [&](const fs_seg &sg, uint32_t rt, uint32_t h, uint32_t slot, uint32_t i_lo, uint32_t i_hi) {
        if (fs_narrow<D, false>(a, sg, sm, rt, h, slot, i_lo, i_hi)) {
            FS_AGAIN(rt, h, slot, i_lo, i_hi);
            fs_narrow<D, true>(a, sg, sm, rt, h, slot, i_lo, i_hi);
        }
    });
}

// The pieces of 32 rows: a lane has 4 dims of a row; the workgroup's four waves share the row's
// pieces, the prefix's and the conversation's, 8 of them in flight each.  What bounds it: the way
// through the launch, the arguments and one load (3.9 us for 8 rows of 128 dims; with a wait for
// every argument 5.7), past some MB of pieces their reading (768 rows of 256 dims, 52 MB: 13.1).
template <int D>
__global__ void __launch_bounds__(256) k_fs_join(fs_join_args a) {
    constexpr uint32_t NP = 8;
    __shared__ __align__(16) float s_x[4][64][4];
    __shared__ float s_m[4][64], s_l[4][64];
    const uint32_t l = threadIdx.x & 63u, w = threadIdx.x >> 6, m2 = l & 31u, h = blockIdx.z, row_b = 32 * blockIdx.x, row = row_b + m2;
    // lane x has conversation x's entries
    const uint32_t t_row0 = a.row0[l], t_rows = a.rows[l], t_pieces = a.pieces[l], t_slot0 = a.slot0[l];
    // (as values: the compiler would load where each is used, one wait after another)
    auto pin = [](uint32_t x) {
        asm volatile("" : "+s"(x));
        return x;
    };
    const uint32_t n_pre = pin(a.pre_pieces), pre_wide = pin(a.pre_wide), n_rows = pin(a.n_rows);
    const bool live = row < n_rows;
    // the first slot of the segment's row r, and from one piece to the next
    auto slots = [&](bool wide, uint32_t slot0, uint32_t pieces, uint32_t rows, uint32_t r, uint32_t &step) {
        const uint32_t gr = wide ? 4u : 1u, rt = r >> (wide ? 7 : 5);
        step = fs_row_tiles(wide, rows) * gr;
        return slot0 + h * pieces * step + rt * gr + (wide ? r >> 5 & 3u : 0u);
    };
    uint32_t step_pre, n_own = 0, step_own = 0, slot_own = 0, r_own = 0;
    const uint32_t slot_pre = slots(pre_wide, 0, n_pre, n_rows, row_b, step_pre);       // (the prefix's rows are all rows)
    // the conversation that the row is in: the last that begins at or before it
    const uint32_t c_lo = __popcll(__builtin_amdgcn_ballot_w64(t_row0 <= row_b)), c_hi = __popcll(__builtin_amdgcn_ballot_w64(t_row0 <= row_b + 31));
    uint32_t cv = c_lo;
    for (uint32_t x = c_lo; x < c_hi; ++x) cv += row >= (uint32_t)__builtin_amdgcn_readlane((int)t_row0, (int)x);
    if (c_hi) {
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_ds_bpermute((int)(4 * (cv ? cv - 1 : 0)), (int)v); };
        const uint32_t row0 = of(t_row0), rows = of(t_rows), pieces = of(t_pieces), slot0 = of(t_slot0);
        if (live && cv && row - row0 < rows) {
            r_own = row - row0;
            n_own = pieces & 0x7fffffffu;
            slot_own = slots(pieces >> 31, slot0, n_own, rows, r_own, step_own);
        }
    }
    const uint32_t n = live ? n_pre + n_own : 0u, t = row / a.G;
    for (uint32_t i = blockIdx.y; i < D / 8; i += gridDim.y) {
        float M = -INFINITY, L = 0.0f;
        kvm_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t q = w; q < n; q += 4 * NP) {
            kvm_u32x4 x[NP];
            kvm_f32x2 ml[NP];
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                const uint32_t k = min(q + 4 * j, n - 1), r = k < n_pre ? m2 : r_own & 31u;
                const uint64_t slot = k < n_pre ? slot_pre + k * step_pre : slot_own + (k - n_pre) * step_own;
                x[j] = *(const kvm_u32x4 *)(a.ws_o + (slot * (D / 8) + i) * 256 + 128 * (l >> 5) + 4 * r);
                ml[j] = *(const kvm_f32x2 *)(a.ws_ml + (slot * 32 + r) * 2);
            }
            float mb = M;
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                if (q + 4 * j >= n) ml[j][0] = -INFINITY;
                mb = fmaxf(mb, ml[j][0]);
            }
            const float top = mb == -INFINITY ? 0.0f : mb, keep = __builtin_amdgcn_exp2f(M - top);
            L *= keep;
            acc *= keep;
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                // (a piece that saw nothing of the row holds anything)
                const float wgt = __builtin_amdgcn_exp2f(ml[j][0] - top);
                const uint32_t has = ml[j][0] == -INFINITY ? 0u : 0xffffffffu;
                L = fmaf(__uint_as_float(__float_as_uint(ml[j][1]) & has), wgt, L);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = fmaf(__uint_as_float(x[j][k] & has), wgt, acc[k]);
            }
            M = mb;
        }
        *(kvm_f32x4 *)s_x[w][l] = acc;
        s_m[w][l] = M;
        s_l[w][l] = L;
        __syncthreads();
        if (w == 0 && live) {
            float mb = M;
#pragma unroll
            for (int j = 1; j < 4; ++j) mb = fmaxf(mb, s_m[j][l]);
            const float top = mb == -INFINITY ? 0.0f : mb;
            L = 0.0f;
            acc = kvm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j) {                 // (a wave without pieces: zeros)
                const float wgt = __builtin_amdgcn_exp2f(s_m[j][l] - top);
                L = fmaf(s_l[j][l], wgt, L);
                acc += *(const kvm_f32x4 *)s_x[j][l] * wgt;
            }
            // nothing visible: zeros
            acc *= L == 0.0f ? 0.0f : 1.0f / L;
            const uint64_t at = ((uint64_t)t * a.n_head + h * a.G + (row - t * a.G)) * D + 8 * i + 4 * (l >> 5);
            if (a.out_type == KVM_TYPE_F32) {
                __builtin_memcpy((float *)a.out + at, &acc, 16);
            } else if (a.out_type == KVM_TYPE_BF16) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                const bf16x4 y = __builtin_convertvector(acc, bf16x4);
                __builtin_memcpy((uint16_t *)a.out + at, &y, 8);
            } else {
                const kvm_f16x4 y = {(_Float16)acc[0], (_Float16)acc[1], (_Float16)acc[2], (_Float16)acc[3]};
                __builtin_memcpy((uint16_t *)a.out + at, &y, 8);
            }
        }
        __syncthreads();
    }
}

// ---- host -----------------------------------------------------------------------
// A step through a window of n tiles that no two of its multiples share a tile with: the
// one from 0.618 n on that has no divisor in common with n.
static uint32_t fs_stride(uint32_t n) {
    auto gcd = [](uint32_t a, uint32_t b) {
        while (b) {
            const uint32_t r = a % b;
            a = b;
            b = r;
        }
        return a;
    };
    uint32_t m = (uint32_t)(0.6180339887 * n);
    m = m ? m : 1;
    while (gcd(m, n) != 1) ++m;
    return m;
}

// The rows from which on a window's units are wide.  An f16 window has nothing to convert: all.
// All figures are of 256 dims; at 128 the rule is the same one, not measured by itself.
// A CU takes a tile of a wide unit of 256 dims in 2.0 us, one of a narrow one in 1.05 (two
// workgroups, 2.1 each): a wide unit pays from three narrow ones' rows on (two's: 48 rows over
// 32,768 cells with 8 x 6 over 2,048, all narrow 30 us, else 28 + 16).  Where some windows stay
// narrow all the same, the wide ones are a launch more (10 us for its start and end) and have to
// save that: 288 rows over 5,003 cells with 16 x 18 over 8,192, all narrow 64 us, else 26 + 52;
// 768 rows over 32,768 with 32 x 24 over 2,048, 251 us and 137 + 35.
static uint32_t fs_wide_rows(const kvm_window *prefix, const kvm_window *const *windows, const uint32_t *n_tokens, uint32_t n_lanes, bool quant,
                             uint32_t n_cu, uint32_t H, uint32_t G, uint32_t n_rows) {
    if (!quant) return 1;
    double saved = 0.0;              // us
    bool narrow = false;
    auto add = [&](const kvm_window *w, uint32_t r) {
        if (!w || !r) return;
        if (r <= 64) narrow = true;
        else saved += (double)(w->n_cells / KVM_TILE_CELLS) * H / n_cu * (1.05 * fs_row_tiles(false, r) - 2.0 * fs_row_tiles(true, r));
    };
    add(prefix, n_rows);
    for (uint32_t i = 0; i < n_lanes; ++i) add(windows ? windows[i] : nullptr, n_tokens[i] * G);
    return narrow && saved < 10.0 ? 0xffffffffu : 65;
}

// Cuts the units of n segments into pieces: of as many tiles at most as let `groups` workgroups at
// a time end first, in tiles, where a piece's start and end cost 4 tiles' time, and no piece is
// below `least`.  Returns that number of tiles.
static uint32_t fs_cut(fs_seg *seg, uint32_t n, bool wide, uint32_t H, uint32_t groups, uint32_t least) {
    uint64_t tiles = 0;
    uint32_t most = 1;
    auto units = [&](uint32_t i) { return (uint64_t)fs_row_tiles(wide, seg[i].n_rows) * H; };
    for (uint32_t i = 0; i < n; ++i) {
        tiles += units(i) * seg[i].n_tiles;
        most = std::max(most, seg[i].n_tiles);
    }
    auto pieces = [&](uint32_t t) {
        uint64_t x = 0;
        for (uint32_t i = 0; i < n; ++i) x += units(i) * ((seg[i].n_tiles + t - 1) / t);
        return x;
    };
    uint32_t best = most;
    uint64_t best_time = ~0ull;
    for (uint32_t rounds = 1; rounds <= 4; ++rounds) {
        // the least number of tiles whose pieces are no more than the rounds' workgroups
        uint32_t lo = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(least, tiles / ((uint64_t)rounds * groups))), hi = most;
        lo = std::max(lo, 1u);
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (pieces(mid) <= (uint64_t)rounds * groups) hi = mid;
            else lo = mid + 1;
        }
        const uint64_t time = (pieces(lo) + groups - 1) / groups * (lo + 4);
        if (time < best_time) {
            best_time = time;
            best = lo;
        }
        if (4 * tiles >= 3ull * groups * lo) break;       // (as even as it gets)
    }
    uint64_t left = 0;
    for (uint32_t i = 0; i < n; ++i) {
        seg[i].pieces = (seg[i].n_tiles + best - 1) / best;
        left += units(i) * seg[i].pieces;
    }
    // The workgroups that are left over shorten the longest pieces (8 lanes x 6 rows over 32,768 +
    // 2,048 cells: 472 pieces of 11 tiles 32.7 us, 512 of 10 and 11 30.0).
    left = (left + groups - 1) / groups * groups - left;
    for (uint32_t x = 0; x < 64 && left; ++x) {
        uint32_t at = n, longest = least;
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t t = (seg[i].n_tiles + seg[i].pieces - 1) / seg[i].pieces;
            if (t > longest && units(i) <= left) at = i, longest = t;
        }
        if (at == n) break;
        const uint32_t p = (seg[at].n_tiles + longest - 2) / (longest - 1);
        const uint64_t more = units(at) * (p - seg[at].pieces);
        if (more > left) break;
        seg[at].pieces = p;
        left -= more;
    }
    return best;
}

// Fills the segments, their pieces and slots.
static int fs_shape(kvm_state *st, const char *what, const kvm_window *prefix, const kvm_window *const *windows,
                    const uint32_t *n_tokens, uint32_t n_lanes, bool quant, uint32_t n_cu, fs_args *a, fs_join_args *j, uint64_t *slots) {
    const uint32_t wide_rows = fs_wide_rows(prefix, windows, n_tokens, n_lanes, quant, n_cu, a->H, a->G, a->n_rows);
    uint32_t n = 0, nw = 0, lane_seg[FS_LANES], own = 0;
    auto add = [&](const kvm_window *w, uint32_t row0, uint32_t n_rows) {
        const uint32_t t = w->n_cells / KVM_TILE_CELLS, m = fs_stride(t);
        const bool iw = n_rows >= wide_rows;
        a->seg[n++] = fs_seg{(const uint8_t *)w->k, (const uint8_t *)w->v, w->cell_pos, t, m, row0, n_rows, (uint32_t)(4ull * (iw ? 8 : 4) * m % t), 1, t, 0};
        if (iw) nw = n;
    };
    if (prefix) add(prefix, 0, a->n_rows);                 // (wide where a conversation is)
    for (int narrow = 0; narrow < 2; ++narrow) {
        uint32_t row = 0;
        own = 0;
        for (uint32_t i = 0; i < n_lanes; ++i) {
            const uint32_t r = n_tokens[i] * a->G;
            if (windows && windows[i] && r) {
                if ((r >= wide_rows) == !narrow) {
                    lane_seg[own] = n;
                    add(windows[i], row, r);
                }
                ++own;
            }
            row += r;
        }
    }
    // Workgroups: what the CUs hold at once.  A tile or more for each wave that has tiles of its
    // own, or half a one where that leaves CUs idle (8 rows over 1,024 + 2 x 256 f16 cells of 2
    // heads: 8.7 us, with 4 tiles a workgroup 15.6; 12 over 1,024 + 2 x 256 q8_0 cells of 4: 2
    // tiles 12.1 us, 4 13.8); a second narrow workgroup a CU for pieces of 4 tiles or more (48 over
    // 4,032 + 4 x 512: 320 workgroups of 2 tiles 19.0, 160 of 4 16.5).
    fs_cut(a->seg, nw, true, a->H, n_cu, 1);
    if (fs_cut(a->seg + nw, n - nw, false, a->H, n_cu, 2) > 4) fs_cut(a->seg + nw, n - nw, false, a->H, 2 * n_cu, 4);
    uint64_t piece = 0, wide = 0;
    for (uint32_t i = 0; i < n; ++i) {
        fs_seg &sg = a->seg[i];
        sg.per = sg.n_tiles / sg.pieces;
        sg.more = sg.n_tiles % sg.pieces;
        a->piece0[i] = (uint32_t)piece;
        piece += (uint64_t)fs_row_tiles(i < nw, sg.n_rows) * a->H * sg.pieces;
        if (i + 1 == nw) wide = piece;
        if (piece > (1u << 24))
            return kvm_fail(st, KVM_ERANGE, "%s: %u rows over these windows are too many for one call", what, a->n_rows);
    }
    for (uint32_t i = n; i < FS_SEGS; ++i) a->piece0[i] = 0xffffffffu;
    a->wide = (uint32_t)wide;
    a->narrow = (uint32_t)(piece - wide);
    *slots = 4 * wide + (piece - wide);
    if (prefix) {
        j->pre_pieces = a->seg[0].pieces;
        j->pre_wide = nw > 0;
    }
    for (uint32_t i = 0; i < FS_LANES; ++i) j->row0[i] = 0xffffffffu;
    for (uint32_t i = 0; i < own; ++i) {
        const uint32_t s = lane_seg[i];
        j->row0[i] = a->seg[s].row0;
        j->rows[i] = a->seg[s].n_rows;
        j->pieces[i] = a->seg[s].pieces | (s < nw ? 0x80000000u : 0u);
        j->slot0[i] = (uint32_t)(s < nw ? 4 * a->piece0[s] : 4 * wide + (a->piece0[s] - wide));
    }
    return KVM_OK;
}

// The most slots of any call of no more tokens and tiles (of all windows), however they are spread
// over conversations.  The slots of a call go up and down with how its units divide into the
// workgroups: 96 tokens over 32,768 f16 cells of 8 heads take 960, 64 tokens and 1 take 1,024.  fs_cut
// makes no more pieces than units, tiles or four rounds of workgroups ask for, in whole rounds.
static uint64_t fs_most_slots(bool quant, uint32_t n_cu, uint32_t H, uint32_t G, uint64_t tokens, uint64_t tiles) {
    const uint64_t rows = tokens * G, lanes = std::min<uint64_t>(tokens, FS_LANES);
    auto pieces = [&](bool wide, uint64_t groups) {
        const uint64_t rt = (rows + fs_unit_rows(wide) - 1) / fs_unit_rows(wide);
        const uint64_t units = (rt + rows / fs_unit_rows(wide) + lanes) * H;       // the prefix's, the conversations'
        return std::min(rt * H * tiles, std::max(4 * groups, (units + groups - 1) / groups * groups));
    };
    return (!quant || rows > 64 ? 4 * pieces(true, n_cu) : 0) + (quant ? pieces(false, 2 * n_cu) : 0);
}

extern "C" int kvm_fa_decode_shared(kvm_state *st, const kvm_window *prefix, const kvm_window *const *windows,
                                    const uint32_t *n_tokens, uint32_t n_lanes, const void *q, int q_type,
                                    const int32_t *q_pos, uint32_t n_head, float scale, int out_type, void *out) {
    const char *what = "fa_decode_shared";
    if (n_lanes == 0) return KVM_OK;
    if (!n_tokens) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    if (n_lanes > FS_LANES) return kvm_fail(st, KVM_ERANGE, "%s: %u lanes > %u", what, n_lanes, FS_LANES);
    if (q_type != KVM_TYPE_F32 && q_type != KVM_TYPE_BF16) return kvm_fail(st, KVM_EUNSUPPORTED, "%s: q type %d", what, q_type);
    if (out_type != KVM_TYPE_F32 && out_type != KVM_TYPE_BF16 && out_type != KVM_TYPE_F16)
        return kvm_fail(st, KVM_EUNSUPPORTED, "%s: output type %d", what, out_type);
    const kvm_window *w0 = prefix;
    uint64_t total = 0, tiles = 0;
    for (uint32_t i = 0; i < n_lanes; ++i) {
        total += n_tokens[i];
        if (!w0 && windows) w0 = windows[i];
    }
    if (!w0) return kvm_fail(st, KVM_EINVAL, "%s: no window", what);
    for (uint32_t i = 0; i <= n_lanes; ++i) {
        const kvm_window *w = i == n_lanes ? prefix : windows ? windows[i] : nullptr;
        if (!w) continue;
        const int rc = kvm_window_check(w);
        if (rc) return kvm_fail(st, rc, "%s: %s %u: bad window", what, i == n_lanes ? "prefix," : "lane", i);
        if (w->n_head_kv != w0->n_head_kv || w->head_dim != w0->head_dim || kvm_k_quant(w->k_type) != kvm_k_quant(w0->k_type))
            return kvm_fail(st, KVM_EUNSUPPORTED, "%s: lane %u: windows of different heads or types", what, i);
        if (((uintptr_t)w->k | (uintptr_t)w->v | (uintptr_t)w->cell_pos) & 15)
            return kvm_fail(st, KVM_EINVAL, "%s: lane %u: a window that is not aligned to 16 bytes", what, i);
        if (w->n_cells / KVM_TILE_CELLS > 65535) return kvm_fail(st, KVM_ERANGE, "%s: lane %u: %u cells", what, i, w->n_cells);
        tiles += w->n_cells / KVM_TILE_CELLS;
    }
    const uint32_t H = w0->n_head_kv, D = w0->head_dim;
    if (n_head == 0 || n_head % H) return kvm_fail(st, KVM_EINVAL, "%s: %u heads on %u", what, n_head, H);
    if (!std::isfinite(scale * 1.4426950408889634f)) return kvm_fail(st, KVM_EINVAL, "%s: scale %g", what, (double)scale);
    if (total > (1u << 24) / (n_head / H)) return kvm_fail(st, KVM_ERANGE, "%s: %llu tokens", what, (unsigned long long)total);
    if (H > 65535) return kvm_fail(st, KVM_ERANGE, "%s: %u kv heads", what, H);
    if (total == 0) return KVM_OK;
    if (!q || !q_pos || !out) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    fs_args a{};
    fs_join_args j{};
    a.H = H;
    a.G = n_head / H;
    a.inv_g = 1.0f / (float)a.G;
    a.n_head = n_head;
    a.n_rows = (uint32_t)total * a.G;
    a.q = q;
    a.q_type = q_type;
    a.q_pos = q_pos;
    j.out = out;
    j.out_type = out_type;
    j.G = a.G;
    j.n_head = n_head;
    j.n_rows = a.n_rows;
    a.q_sign = scale < 0.0f ? -1.0f : scale > 0.0f ? 1.0f : 0.0f;
    a.c = scale != 0.0f ? fabsf(scale) * 1.4426950408889634f : 1.0f;
    uint64_t slots = 0;
    const bool quant = kvm_k_quant(w0->k_type);
    const int rc = fs_shape(st, what, prefix, windows, n_tokens, n_lanes, quant, st ? st->n_cu : 256u, &a, &j, &slots);
    if (rc) return rc;
    if (!st) return KVM_EINVAL;
    const size_t slot_bytes = 32 * (D * 4 + 8), bytes_o = (size_t)slots * 32 * D * 4;
    KVM_HIP(st, hipSetDevice(st->device));
    if (slots) {
        void *ws = nullptr;
        const uint64_t most = fs_most_slots(quant, st->n_cu, H, a.G, total, tiles);
        if (const int bad = kvm_shared_workspace(st, what, slots * slot_bytes, most * slot_bytes, &ws)) return bad;
        a.ws_o = (float *)ws;
        a.ws_ml = (float *)((uint8_t *)a.ws_o + bytes_o);
        j.ws_o = a.ws_o;
        j.ws_ml = a.ws_ml;
    }
    // a workgroup of the join has 8 dims, or more of them where all CUs have two all the same
    // (its start is most of its work: 768 rows of 256 dims, 15.6 us by 8 dims)
    const uint64_t blocks = (uint64_t)kvm_cdiv(a.n_rows, 32) * H;
    uint32_t by = D / 8;
    while (by > 1 && blocks * by >= 4ull * st->n_cu) by /= 2;
    auto go = [&](auto d, auto qt) {
        constexpr int DD = decltype(d)::value;
        constexpr bool Q = decltype(qt)::value;
        auto grid = [](uint32_t n) { return dim3(n < 8 ? n : (n + 7) / 8 * 8); };       // (a grid of 8 for each XCD's)
        if (a.wide) hipLaunchKernelGGL((k_fs_wide<DD, Q>), grid(a.wide), dim3(512), 0, st->stream, a);
        if (Q && a.narrow) hipLaunchKernelGGL((k_fs_narrow<DD>), grid(a.narrow), dim3(256), 0, st->stream, a);
        hipLaunchKernelGGL((k_fs_join<DD>), dim3(kvm_cdiv(a.n_rows, 32), by, H), dim3(256), 0, st->stream, j);
    };
    auto go_d = [&](auto d) {
        if (quant) go(d, std::true_type{});
        else go(d, std::false_type{});
    };
    if (D == 256) go_d(std::integral_constant<int, 256>{});
    else go_d(std::integral_constant<int, 128>{});
    KVM_LAUNCH_CHECK(st, what);
    return KVM_OK;
}
