// kvm_fa_shared.hip -- decode / verify attention of several conversations that share a
// long prefix (kvm_fa_decode_shared): every query attends over the prefix window's cells
// and its own conversation's, one softmax over both.
//
//   o_t = sum_c p_tc v_c / sum_c p_tc, p_tc = exp(scale q_t . k_c - m_t) over the cells c of
//   both windows with 0 <= position <= the query's
//
// splits over any parts of the cells into (m, l, o) of each part, joined by the parts'
// maxima.  A part is a piece: some tiles of one window for at most 32 rows of a kv head (a
// row is a token and a query head of the group).  The prefix's rows are all conversations'
// tokens side by side, so its keys and values are read, and brought to f16, once for 32
// rows; a conversation's own window is one for its rows.  k_fs_attn forms the pieces,
// k_fs_join joins those of each row.
//
// A workgroup is 4 waves, one a SIMD; each takes every fourth of the piece's tiles, for all
// its rows, so that nothing is shared in the loop and no barrier is in it: tiles go from
// memory into registers (the tile layout is the matrix operands'), a half tile's registers
// are loaded for the next tile as soon as they are used.  S^T = K Q^T and O^T += V^T P^T on
// 32x32x16 f16 MFMAs; Q is in LDS as operands.  Quantised tiles become f16 on the way: K and
// V as (f16)(q d), Q and P rounded to f16, everything else fp32.  Key order: score row i of a
// half tile is key i with bits 2 and 3 swapped, so that a lane's scores are 8 consecutive
// keys of each 16, what the P V operand wants.  The waves' sums meet in LDS at the end.
//
// The tiles of all units (32 rows of a head over one window) are dealt to the workgroups in
// equal shares, in an order that steps through a window in strides: a
// part-filled window's live tiles are spread evenly over its pieces.
#include "kvm_f16_dev.h"

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
};

struct fs_args {
    const void *q;
    const int32_t *q_pos;
    void *out;
    float *ws_o;                 // pieces [slot][dim / 8][lane][4]
    float *ws_ml;                // [slot][row][2]: scaled maximum, sum
    uint32_t H, G, n_head, n_rows;
    uint32_t n_seg, log_p;       // workgroups: 1 << log_p
    float c, q_sign;             // |scale| log2(e); q times -1 for a negative scale, and 0 (c = 1) for none
    int q_type, out_type;
    uint32_t has_prefix;         // segment 0 is the prefix
    uint32_t tile0[FS_SEGS + 1]; // tiles of the units of the segments before
    uint32_t unit0[FS_SEGS];     // units before
    uint32_t lane0[FS_LANES];    // first row of the conversations' segments, the rest ~0
    fs_seg seg[FS_SEGS];
};
static_assert(sizeof(fs_args) <= 4096, "kernel arguments");

__host__ __device__ inline uint32_t fs_row_tiles(uint32_t n_rows) { return (n_rows + 31) / 32; }
// Workgroup p has tiles [fs_share(p), fs_share(p + 1)) of the units' after each other.
__host__ __device__ inline uint32_t fs_share(uint32_t tiles, uint32_t log_p, uint32_t p) { return (uint32_t)((uint64_t)p * tiles >> log_p); }
// The workgroup whose share holds tile x.
__host__ __device__ inline uint32_t fs_owner(uint32_t tiles, uint32_t log_p, uint32_t x) {
    const uint32_t n = 1u << log_p;
    uint32_t p = (uint32_t)((float)x * ((float)n / (float)tiles));
    p = p < n ? p : n - 1;
    while (p > 0 && fs_share(tiles, log_p, p) > x) --p;
    while (p + 1 < n && fs_share(tiles, log_p, p + 1) <= x) ++p;
    return p;
}

// Workgroups of a CU: the f16 tiles of 256 dims take the registers of two waves.
__host__ __device__ constexpr uint32_t fs_resident(uint32_t D, bool quant) { return D == 256 && !quant ? 1 : 2; }

template <int D, bool QUANT>
struct fs_geo {
    static constexpr int KS = D / 16, NB = D / 32, DT = D / 32;              // k-steps, 32-dim blocks, dim tiles
    static constexpr int DW = DT / 4;                     // dim tiles that a wave adds up at the end
    static constexpr uint32_t KB = QUANT ? 64u * D + 128u * NB : 128u * D, VB = QUANT ? 32u * D + 128u * NB : 128u * D;
    static constexpr int KH = QUANT ? NB : 2 * NB;        // 16-byte loads of a half tile's K
    static constexpr int SETS = D == 256 ? 1 : 2;                  // half tiles of K (and f16 V) in registers
    static constexpr uint32_t QU = 528;                   // LDS bytes of a unit of Q: 8 dims of 32 rows, 16 bytes apart in the banks
};

template <int D, bool QUANT>
struct fs_lds {
    using G = fs_geo<D, QUANT>;
    alignas(16) uint8_t q[2 * G::KS * G::QU];
    alignas(16) uint8_t sc[4][2][QUANT ? 2 : 1][QUANT ? 1024 : 16];           // a wave's tile and its next: K scales, V scales
    alignas(16) int32_t cp[4][2][64];                     // and their cells' positions
    alignas(16) float x[4][G::DW * 4 * 256];              // chunks of O on their way
    float ml[4][2][32];
    uint32_t odd[4][2];
    uint32_t list[FS_BATCH];
    uint8_t flag[FS_BATCH];
};

// x, from which the compiler cannot tell that a value formed of it does not change in a
// loop: hoisted, lane addresses take the registers that the accumulators need.
__device__ __forceinline__ uint32_t fs_opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
// K row i of a half tile is this key: bits 2 and 3 swapped.
__device__ __forceinline__ uint32_t fs_key(uint32_t i) { return (i & 0x13) | (i & 4) << 1 | (i & 8) >> 1; }

// Nothing moves over it.
#define FS_FENCE() __builtin_amdgcn_sched_barrier(0)

// A piece: tiles [i_lo, i_hi) in the unit's order.
template <int D, bool QUANT>
__device__ __forceinline__ void fs_piece(const fs_args &a, const fs_seg &sg, fs_lds<D, QUANT> &sm, uint32_t rt, uint32_t h, uint32_t slot,
                                         uint32_t i_lo, uint32_t i_hi) {
    using G = fs_geo<D, QUANT>;
    constexpr int KS = G::KS, NB = G::NB, DT = G::DT, DW = G::DW, KH = G::KH, SETS = G::SETS;
    constexpr uint32_t KB = G::KB, VB = G::VB, QU = G::QU;
    const uint32_t tid = threadIdx.x, l = tid & 63u, g2 = l >> 5, m2 = l & 31u;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t rows = min(32u, sg.n_rows - 32 * rt), row_g = sg.row0 + 32 * rt;

    // ---- the rows: Q as f16 operands in LDS, the rows' limits
    for (uint32_t x = tid; x < 32u * 2 * KS; x += 256) {
        // 8 rows x 8 units an instruction
        const uint32_t b = x >> 6, r = b % 4 * 8 + (x & 63u) / 8, u = b / 4 * 8 + (x & 7u);
        float v[8];
        if (r < rows) {
            const uint32_t t = (row_g + r) / a.G;
            const uint64_t e = ((uint64_t)t * a.n_head + h * a.G + (row_g + r - t * a.G)) * D + 8 * u;
            if (a.q_type == KVM_TYPE_F32) {
                __builtin_memcpy(v, (const float *)a.q + e, 32);
            } else {
                kvm_u32x4 y;
                __builtin_memcpy(&y, (const uint16_t *)a.q + e, 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(j & 1 ? y[j >> 1] & 0xffff0000u : y[j >> 1] << 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        }
        kvm_f16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (_Float16)(v[j] * a.q_sign);
        *(kvm_f16x8 *)(sm.q + u * QU + r * 16) = o;
    }
    const int32_t qp = m2 < rows ? a.q_pos[(row_g + m2) / a.G] : -1;
    const uint32_t qlim = qp >= 0 ? (uint32_t)qp + 1u : 0u;      // a cell is visible iff (unsigned)position < qlim
    const uint32_t all_lim = kvm_wave_min_u32(m2 < rows ? qlim : 0xffffffffu), some_lim = ~kvm_wave_min_u32(~qlim);

    kvm_f32x16 O[DT];
    float ms = -INFINITY, lp = 0.0f;     // the row's reference maximum (times c), the lane's share of its sum
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] = 0.0f;

    // operand addresses of a lane
    const uint32_t key = fs_key(m2);
    const uint32_t k_lane = ((key >> 4) * (QUANT ? NB / 2 : NB) * 64 + 16 * g2 + (key & 15)) * 16;
    const uint32_t v_lane = ((m2 >> 4) * 64 + 16 * g2 + (m2 & 15)) * (QUANT ? 8 : 32);
    const uint8_t *const k_head = sg.k + (uint64_t)h * sg.n_tiles * KB, *const v_head = sg.v + (uint64_t)h * sg.n_tiles * VB;

    for (uint32_t b0 = i_lo; b0 < i_hi; b0 += FS_BATCH) {
        // ---- the batch's tiles that some row sees; bit 31: every cell visible to every row
        const uint32_t nb = min(FS_BATCH, i_hi - b0);
        auto tile_of = [&](uint32_t i) { return (b0 + i) * sg.mult % sg.n_tiles; };     // (n_tiles < 2^16)
        for (uint32_t r0 = 0; r0 < nb; r0 += 64) {
            kvm_u32x4 c[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t i = r0 + 16 * r + 4 * w + (l >> 4);
                c[r] = *(const kvm_u32x4 *)(sg.cell_pos + (uint64_t)tile_of(i < nb ? i : 0u) * 64 + 4 * (l & 15));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t i = r0 + 16 * r + 4 * w + (l >> 4);
                const uint32_t least = min(min(c[r][0], c[r][1]), min(c[r][2], c[r][3])), most = max(max(c[r][0], c[r][1]), max(c[r][2], c[r][3]));
                const uint32_t some = (uint32_t)(__builtin_amdgcn_ballot_w64(least < some_lim) >> (l & 48)) & 0xffffu;
                const uint32_t all = (uint32_t)(__builtin_amdgcn_ballot_w64(most < all_lim) >> (l & 48)) & 0xffffu;
                if (i < nb && (l & 15) == 0) sm.flag[i] = (uint8_t)((some != 0) | (all == 0xffffu) << 1);
            }
        }
        __syncthreads();                                  // flags, and Q
        uint32_t n_t = 0;
#pragma unroll
        for (uint32_t x = 0; x < FS_BATCH / 64; ++x) {
            const uint32_t f = 64 * x + l < nb ? sm.flag[64 * x + l] : 0u;
            const uint64_t bal = __builtin_amdgcn_ballot_w64(f & 1u);
            const uint32_t rank = n_t + __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0u));
            if ((f & 1u) && (int)x == w) sm.list[rank] = tile_of(64 * x + l) | (f >> 1) << 31;
            n_t += __popcll(bal);
        }
        n_t = __builtin_amdgcn_readfirstlane(n_t);
        __syncthreads();

        // ---- the wave's tiles: list entries w, w + 4, ..  Registers of a half tile are
        // loaded for the next tile where this one's are used up.
        kvm_u32x4 kr[SETS][KH], vh[QUANT ? 1 : SETS][QUANT ? 1 : 2 * DT];
        uint32_t vq[QUANT ? 2 * DT : 1];                  // quantised V of a half tile
        // (past the wave's last tile the bounds let nothing through)
        auto rsrc = [&](const void *head, uint32_t e, uint32_t bytes, bool more) {
            return __builtin_amdgcn_make_buffer_rsrc((void *)((const uint8_t *)head + (uint64_t)(e & 0x7fffffffu) * bytes), (short)0, more ? bytes : 0u, 0x00020000);
        };
        auto load_k = [&](__amdgpu_buffer_rsrc_t r, int half) {
#pragma unroll
            for (int i = 0; i < KH; ++i)
                kr[half % SETS][i] = __builtin_amdgcn_raw_buffer_load_b128(r, k_lane + (i & 1) * 512, half * (QUANT ? NB : 2 * NB) * 1024 + (i >> 1) * 1024, 0);
        };
        auto load_v = [&](__amdgpu_buffer_rsrc_t r, int half) {
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                if constexpr (QUANT) vq[i] = __builtin_amdgcn_raw_buffer_load_b32(r, v_lane + (i & 1) * 256 + half * 4, (i >> 1) * 1024, 0);
                else vh[half % SETS][i] = __builtin_amdgcn_raw_buffer_load_b128(r, v_lane + (i & 1) * 1024 + half * 16, (i >> 1) * 4096, 0);
            }
        };
        // Scales and positions go to LDS by direct copies (lane l writes 16 or 4 bytes at M0 +
        // 16 l or 4 l), issued from asm, so that the compiler adds no wait for them; the asm
        // restores M0, which the compiler reserves.
        auto copy16 = [&](const uint8_t *src, void *dst) {
            const uint32_t off = 16u * (fs_opaque(l) & (D == 256 ? 63u : 31u));   // (128 dims: 512 bytes of scales)
            uint32_t m0_saved;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                         : "=&s"(m0_saved) : "v"(off), "s"((uint32_t)(uintptr_t)(fs_lds_ptr)dst), "s"(src) : "memory");
        };
        auto copies = [&](uint32_t e, uint32_t buf) {
            const uint32_t t = e & 0x7fffffffu;
            if constexpr (QUANT) {
                copy16(k_head + (uint64_t)t * KB + 64 * D, sm.sc[w][buf][0]);
                copy16(v_head + (uint64_t)t * VB + 32 * D, sm.sc[w][buf][1]);
            }
            uint32_t m0_saved;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %3\n\ts_mov_b32 m0, %0"
                         : "=&s"(m0_saved) : "v"(4u * fs_opaque(l)), "s"((uint32_t)(uintptr_t)(fs_lds_ptr)&sm.cp[w][buf][0]), "s"(sg.cell_pos + (uint64_t)t * 64) : "memory");
        };
        // keys base .. base + 7 of the lanes' bits, together
        auto gather = [&](uint32_t base, uint32_t bits) {
            if (l < 2) sm.odd[w][l] = 0;
            __builtin_amdgcn_wave_barrier();
            if (bits) atomicOr(&sm.odd[w][base >> 5], bits << (base & 31u));
            __builtin_amdgcn_wave_barrier();
            return (uint64_t)__builtin_amdgcn_readfirstlane(sm.odd[w][1]) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane(sm.odd[w][0]);
        };
        uint32_t e = 0;
        if ((uint32_t)w < n_t) {
            e = __builtin_amdgcn_readfirstlane(sm.list[w]);
            const auto rk = rsrc(k_head, e, KB, true), rv = rsrc(v_head, e, VB, true);
            copies(e, 0);
            load_k(rk, 0);
            if (SETS == 2) load_k(rk, 1);
            load_v(rv, 0);
            if (!QUANT && SETS == 2) load_v(rv, 1);
        }
        uint32_t buf = 0;
        for (uint32_t j = w; j < n_t; j += 4, buf ^= 1) {
            // the tile's copies: the first tile's half tiles, or more, were loaded after them
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"(SETS * KH + (QUANT ? 1 : SETS) * 2 * DT) : "memory");
            const bool more = j + 4 < n_t;
            const uint32_t en = __builtin_amdgcn_readfirstlane(sm.list[more ? j + 4 : j]);
            const auto rk = rsrc(k_head, en, KB, more), rv = rsrc(v_head, en, VB, more);
            const bool full = e >> 31;
            // keys that some row sees; those of them that not all do and whose value is no
            // finite number
            uint64_t seen = ~0ull, part = 0, odd = 0;
            if (!full) {
                asm volatile("" ::: "memory");            // keep it on this (rare) path
                const uint32_t cp = (uint32_t)sm.cp[w][buf][fs_opaque(l)];
                seen = __builtin_amdgcn_ballot_w64(cp < some_lim);
                part = seen & ~__builtin_amdgcn_ballot_w64(cp < all_lim);
                if constexpr (QUANT) {
                    // What no row sees counts nothing, whatever it holds: a scale of 0.  (Lane
                    // l has the scales of 8 keys of a block.)
                    const uint32_t lo = fs_opaque(l), base = 32 * (lo >> 2 & 1u) + 8 * (lo & 3u), on = (uint32_t)(seen >> base) & 0xffu, pt = (uint32_t)(part >> base) & 0xffu;
                    kvm_u32x4 scv = *(const kvm_u32x4 *)(sm.sc[w][buf][1] + 16 * lo);
                    uint32_t bad = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t sh = 16 * (i & 1), v = scv[i >> 1] >> sh & 0xffffu;
                        if (lo < 8u * NB && (pt >> i & 1u) && (v & 0x7c00u) == 0x7c00u) bad |= 1u << i;
                        if (!(on >> i & 1u) || (bad >> i & 1u)) scv[i >> 1] &= ~(0xffffu << sh);
                    }
                    *(kvm_u32x4 *)(sm.sc[w][buf][1] + 16 * lo) = scv;
                    if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) odd = gather(base, bad);
                }
            }
            if (more) copies(en, buf ^ 1);

#pragma unroll
            for (int half = 0; half < 2; ++half) {
                // ---- S^T of 32 keys: K operand i + 1 is made while the MFMA of i runs; what
                // comes from LDS is read two steps ahead
                kvm_f32x16 S;
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] = 0.0f;
                uint32_t ksc[NB];                         // the scales of the lane's key
                if constexpr (QUANT) {
                    const uint32_t k = fs_key(fs_opaque(l) & 31u);
#pragma unroll
                    for (int b = 0; b < NB; ++b) ksc[b] = *(const uint16_t *)(sm.sc[w][buf][0] + ((2 * half + (k >> 4)) * NB + b) * 32 + 2 * (k & 15));
                }
                const uint8_t *const sq = sm.q + g2 * QU + m2 * 16;
                // operands in the order of the K loads: (block pair, 16-dim half | block of the pair)
                auto ks_of = [](int i) { return QUANT ? 4 * (i >> 2) + 2 * (i & 1) + (i >> 1 & 1) : i; };
                auto k_op = [&](int i) {
                    if constexpr (QUANT) {
                        const kvm_u32x4 x = kr[half % SETS][i >> 1];
                        return pf_q8(x[2 * (i & 1)], x[2 * (i & 1) + 1], ksc[2 * (i >> 2) + (i & 1)]);
                    } else {
                        return __builtin_bit_cast(kvm_f16x8, kr[half % SETS][i]);
                    }
                };
                auto q_op = [&](int i) { return *(const kvm_f16x8 *)(sq + 2 * ks_of(i) * QU); };
                kvm_f16x8 kop = k_op(0), qr[3] = {q_op(0), q_op(1)};
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    if (i + 2 < KS) qr[(i + 2) % 3] = q_op(i + 2);
                    FS_FENCE();
                    S = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, qr[i % 3], S, 0, 0, 0);
                    if (i + 1 < KS) kop = k_op(i + 1);
                    FS_FENCE();
                }
                if (SETS == 2) load_k(rk, half);
                else if (half == 0) load_k(rsrc(k_head, e, KB, true), 1);
                else load_k(rk, 0);

                // ---- softmax: P as f16 operands
                if (!full) {
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const kvm_u32x4 x = *(const kvm_u32x4 *)(&sm.cp[w][buf][32 * half + 16 * (i >> 1) + 8 * (fs_opaque(l) >> 5) + 4 * (i & 1)]);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!(x[r] < qlim)) S[4 * i + r] = -INFINITY;
                    }
                }
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
                if constexpr (!QUANT) {
                    if (!full) {
                        // values of keys that no row sees become 0
                        asm volatile("" ::: "memory");
                        uint32_t bad[2] = {0, 0};
#pragma unroll
                        for (int i = 0; i < 2 * DT; ++i) {
                            const uint32_t base = 32 * half + 16 * (i & 1) + 8 * g2;
                            const uint32_t on = (uint32_t)(seen >> base) & 0xffu, pt = (uint32_t)(part >> base) & 0xffu;
                            kvm_u32x4 &v = vh[half % SETS][i];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const uint32_t sh = 16 * (k & 1);
                                const bool no = (pt >> k & 1u) && (v[k >> 1] >> sh & 0x7c00u) == 0x7c00u;
                                if (no) bad[i & 1] |= 1u << k;
                                if (!(on >> k & 1u) || no) v[k >> 1] &= ~(0xffffu << sh);
                            }
                        }
                        if (__builtin_amdgcn_ballot_w64((bad[0] | bad[1]) != 0) != 0)
                            odd |= gather(32 * half + 8 * g2, bad[0] | bad[1] << 16);
                    }
                }
                kvm_u32x4 vs[3];
                auto v_scale = [&](int i) {
                    if constexpr (QUANT) vs[i % 3] = *(const kvm_u32x4 *)(sm.sc[w][buf][1] + (((i >> 1) * 2 + half) * 4 + 2 * (i & 1) + g2) * 16);
                };
                auto v_op = [&](int i) {
                    if constexpr (QUANT) return pf_q4(vq[i], vs[i % 3]);
                    else return __builtin_bit_cast(kvm_f16x8, vh[half % SETS][i]);
                };
                v_scale(0);
                v_scale(1);
                kvm_f16x8 vop = v_op(0);
#pragma unroll
                for (int i = 0; i < 2 * DT; ++i) {
                    if (i + 2 < 2 * DT) v_scale(i + 2);
                    FS_FENCE();
                    O[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop, pb[i & 1], O[i >> 1], 0, 0, 0);
                    if (i + 1 < 2 * DT) vop = v_op(i + 1);
                    FS_FENCE();
                }
                if ((uint32_t)(odd >> (32 * half)) != 0) {
                    // A value that is no finite number, at a key that some rows see and others
                    // do not: 0 times it is not 0.  The product took 0 for it; here it is added
                    // where p is not 0 (p times it is itself).
                    asm volatile("" : "+v"(pb[0]), "+v"(pb[1]) : : "memory");     // keep it on this (rare) path
                    const uint8_t *const v_tile = v_head + (uint64_t)(e & 0x7fffffffu) * VB;
                    float *const sx = sm.x[w];
                    for (uint32_t k = 0; k < 32; ++k) {
                        const uint32_t c = 32 * half + k, lo = fs_opaque(l);
                        if (!(odd >> c & 1u)) continue;
                        // the key's values that are not finite, and where its p are not 0
#pragma unroll
                        for (uint32_t d = lo; d < D; d += 64) {
                            float v;
                            if constexpr (QUANT)
                                v = (float)((int)(v_tile[kvm_vq_byte(c, d)] >> kvm_vq_shift(c) & 15u) - 8) * kvm_h2f(*(const uint16_t *)(v_tile + kvm_vd_off(D, c, d / 32)));
                            else v = kvm_h2f(((const uint16_t *)v_tile)[kvm_vh_idx(c, d)]);
                            sx[d] = v - v == 0.0f ? 0.0f : v;
                        }
                        bool has = false;
#pragma unroll
                        for (uint32_t r = 0; r < 16; ++r) has |= lo >> 5 == (k >> 3 & 1u) && r == (k >> 4) * 8 + (k & 7u) && !((float)pb[r >> 3][r & 7] == 0.0f);
                        const uint64_t b = __builtin_amdgcn_ballot_w64(has);
                        const bool mine = ((uint32_t)b | (uint32_t)(b >> 32)) >> (lo & 31u) & 1u;
                        __builtin_amdgcn_wave_barrier();
#pragma unroll
                        for (int x = 0; x < 4 * DT; ++x) {
                            const kvm_f32x4 v = *(const kvm_f32x4 *)(sx + 8 * x + 4 * (lo >> 5));
#pragma unroll
                            for (int r = 0; r < 4; ++r) O[x >> 2][4 * (x & 3) + r] += mine ? v[r] : 0.0f;
                            FS_FENCE();
                        }
                        __builtin_amdgcn_wave_barrier();
                    }
                }
                if (!QUANT && SETS == 2) load_v(rv, half);
                else if (half == 0) load_v(rsrc(v_head, e, VB, true), 1);
                else load_v(rv, 0);
            }
            e = en;
        }
        __syncthreads();                                  // the next batch's flags and list
    }

    // ---- the waves' sums: one maximum, then chunk by chunk to the wave that adds it up
    const float lr = kvm_add_xor32(lp);
    if (g2 == 0) {
        sm.ml[w][0][m2] = ms;
        sm.ml[w][1][m2] = lr;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sm.ml[0][0][m2], sm.ml[1][0][m2]), fmaxf(sm.ml[2][0][m2], sm.ml[3][0][m2]));
    float L = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) L += sm.ml[x][0][m2] == -INFINITY ? 0.0f : sm.ml[x][1][m2] * __builtin_amdgcn_exp2f(sm.ml[x][0][m2] - M);
    const float wgt = __builtin_amdgcn_exp2f(ms - M);
    // quad i of O: dims 8 i + 4 g2 .. + 3 of the lane's row, weighted
    auto quad = [&](int i) {
        kvm_f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ms == -INFINITY ? 0.0f : O[i >> 2][4 * (i & 3) + k] * wgt;
        return v;
    };
    constexpr int NQ = DW * 4;                            // quads of a chunk
    kvm_f32x4 acc[NQ];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (q == w) {
#pragma unroll
            for (int x = 0; x < NQ; ++x) acc[x] = quad(q * NQ + x);
        }
    for (int round = 1; round < 4; ++round) {
        const int to = (w + round) & 3;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q == to) {
#pragma unroll
                for (int x = 0; x < NQ; ++x) *(kvm_f32x4 *)(sm.x[q] + 256 * x + 4 * l) = quad(q * NQ + x);
            }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < NQ; ++x) acc[x] += *(const kvm_f32x4 *)(sm.x[w] + 256 * x + 4 * l);
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) *(kvm_f32x4 *)(a.ws_o + ((uint64_t)slot * (D / 8) + w * NQ + x) * 256 + 4 * l) = acc[x];
    if (w == 0 && g2 == 0) {
        float *ml = a.ws_ml + ((uint64_t)slot * 32 + m2) * 2;
        ml[0] = M;
        ml[1] = L;
    }
}

template <int D, bool QUANT>
__global__ void __launch_bounds__(256, fs_resident(D, QUANT)) k_fs_attn(fs_args a) {
    __shared__ fs_lds<D, QUANT> sm;
    const uint32_t tid = threadIdx.x, l = tid & 63u;
    // neighbouring shares on one XCD: their units read the same tiles
    uint32_t p = blockIdx.x;
    if (a.log_p >= 3) p = (p & 7u) << (a.log_p - 3) | p >> 3;
    const uint32_t tiles = a.tile0[a.n_seg], lo = fs_share(tiles, a.log_p, p), hi = fs_share(tiles, a.log_p, p + 1);
    uint32_t s = __popcll(__builtin_amdgcn_ballot_w64(l < a.n_seg && a.tile0[l < a.n_seg ? l : 0u] <= lo)) - 1;
    if (a.n_seg > 64 && a.tile0[64] <= lo) s = 64;
    s = __builtin_amdgcn_readfirstlane(s);
    for (uint32_t at = lo; at < hi;) {
        const fs_seg &sg = a.seg[s];
        const uint32_t n_rt = fs_row_tiles(sg.n_rows), ul = (at - a.tile0[s]) / sg.n_tiles, t0 = a.tile0[s] + ul * sg.n_tiles;
        fs_piece<D, QUANT>(a, sg, sm, ul % n_rt, ul / n_rt, p + a.unit0[s] + ul, at - t0, min(hi - t0, sg.n_tiles));
        at = t0 + sg.n_tiles;
        if (at >= a.tile0[s + 1]) ++s;
    }
}

// The pieces of 32 rows' 8 dims: a lane has 4 dims of a row; the workgroup's four waves share
// the prefix's pieces, wave 0 also takes the conversation's.
template <int D, int NP>
__global__ void __launch_bounds__(256) k_fs_join(fs_args a) {
    const uint32_t l = threadIdx.x & 63u, w = threadIdx.x >> 6, m2 = l & 31u, i = blockIdx.y, h = blockIdx.z, row = 32 * blockIdx.x + m2;
    const uint32_t tiles = a.tile0[a.n_seg];
    float M = -INFINITY, L = 0.0f;
    kvm_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    // pieces first, first + step, .. of unit ul of segment s; r: the row in the unit
    auto take = [&](uint32_t s, uint32_t ul, uint32_t r, uint32_t first, uint32_t step, bool live) {
        const fs_seg &sg = a.seg[s];
        const uint32_t t0 = a.tile0[s] + ul * sg.n_tiles;
        const uint32_t q0 = fs_owner(tiles, a.log_p, t0), q1 = fs_owner(tiles, a.log_p, t0 + sg.n_tiles - 1);
        const uint64_t u = a.unit0[s] + ul;
        for (uint32_t q = q0 + first; q <= q1; q += step * NP) {
            kvm_f32x4 x[NP];
            float m[NP], sum[NP];
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                const uint64_t slot = min(q + step * j, q1) + u;
                x[j] = *(const kvm_f32x4 *)(a.ws_o + (slot * (D / 8) + i) * 256 + 128 * (l >> 5) + 4 * r);
                const kvm_f32x2 ml = *(const kvm_f32x2 *)(a.ws_ml + (slot * 32 + r) * 2);
                m[j] = live && q + step * j <= q1 ? ml[0] : -INFINITY;
                sum[j] = ml[1];
            }
            float mb = M;
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) mb = fmaxf(mb, m[j]);
            const float keep = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mb);
            L *= keep;
            acc *= keep;
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                // (a piece that saw nothing, or is not the lane's, holds anything)
                const float wgt = __builtin_amdgcn_exp2f(m[j] - mb);
                const bool no = m[j] == -INFINITY;
                L += no ? 0.0f : sum[j] * wgt;
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] += no ? 0.0f : x[j][k] * wgt;
            }
            M = mb;
        }
    };
    const bool live = row < a.n_rows;
    if (a.has_prefix) {
        // the prefix's rows are all rows
        const uint32_t n_rt = fs_row_tiles(a.n_rows);
        take(0, h * n_rt + blockIdx.x, m2, w, 4, live);
    }
    if (w == 0) {
        // the conversation that the row is in
        uint32_t s = 0;
#pragma unroll
        for (uint32_t x = 0; x < FS_LANES; ++x) s += row >= a.lane0[x];
        const bool own = live && s > 0 && row < a.seg[a.has_prefix + s - 1].row0 + a.seg[a.has_prefix + s - 1].n_rows;
        if (own) {
            const uint32_t x = a.has_prefix + s - 1, r = row - a.seg[x].row0;
            take(x, h * fs_row_tiles(a.seg[x].n_rows) + r / 32, r % 32, 0, 1, true);
        }
    }
    __shared__ __align__(16) float s_x[4][64][4];
    __shared__ float s_m[4][64], s_l[4][64];
    *(kvm_f32x4 *)s_x[w][l] = acc;
    s_m[w][l] = M;
    s_l[w][l] = L;
    __syncthreads();
    if (w != 0 || !live) return;
    float mb = M;
#pragma unroll
    for (int j = 1; j < 4; ++j) mb = fmaxf(mb, s_m[j][l]);
    L = 0.0f;
    acc = kvm_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool no = s_m[j][l] == -INFINITY;
        const float wgt = __builtin_amdgcn_exp2f(s_m[j][l] - mb);
        L += no ? 0.0f : s_l[j][l] * wgt;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += no ? 0.0f : s_x[j][l][k] * wgt;
    }
    // nothing visible: zeros
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint32_t t = row / a.G;
    const uint64_t at = ((uint64_t)t * a.n_head + h * a.G + (row - t * a.G)) * D + 8 * i + 4 * (l >> 5);
    acc *= inv;
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

// Fills the segments, their tiles and the number of workgroups.
static int fs_shape(kvm_state *st, const char *what, const kvm_window *prefix, const kvm_window *const *windows,
                    const uint32_t *n_tokens, uint32_t n_lanes, uint32_t n_wg, fs_args *a, uint32_t *units) {
    uint64_t unit = 0, tiles = 0;
    uint32_t n = 0;
    auto add = [&](const kvm_window *w, uint32_t row0, uint32_t n_rows) {
        const uint32_t t = w->n_cells / KVM_TILE_CELLS;
        a->tile0[n] = (uint32_t)tiles;
        a->unit0[n] = (uint32_t)unit;
        a->seg[n++] = fs_seg{(const uint8_t *)w->k, (const uint8_t *)w->v, w->cell_pos, t, fs_stride(t), row0, n_rows};
        const uint64_t u = (uint64_t)fs_row_tiles(n_rows) * a->H;
        unit += u;
        tiles += u * t;
    };
    a->has_prefix = prefix && a->n_rows;
    if (a->has_prefix) add(prefix, 0, a->n_rows);
    uint32_t row = 0, own = 0;
    for (uint32_t i = 0; i < FS_LANES; ++i) a->lane0[i] = 0xffffffffu;
    for (uint32_t i = 0; i < n_lanes; ++i) {
        const uint32_t r = n_tokens[i] * a->G;
        if (windows && windows[i] && r) {
            a->lane0[own++] = row;
            add(windows[i], row, r);
        }
        row += r;
    }
    if (tiles > 0x7fffffffu || unit > (1u << 24))
        return kvm_fail(st, KVM_ERANGE, "%s: %u rows over these windows are too many for one call", what, a->n_rows);
    a->tile0[n] = (uint32_t)tiles;
    a->n_seg = n;
    // a share of four tiles at least: one a wave
    a->log_p = 0;
    while ((2u << a->log_p) <= n_wg && (8ull << a->log_p) <= tiles) ++a->log_p;
    *units = (uint32_t)unit;
    return KVM_OK;
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
    uint64_t total = 0;
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
        if (w->n_cells / KVM_TILE_CELLS > 65535) return kvm_fail(st, KVM_ERANGE, "%s: lane %u: %u cells", what, i, w->n_cells);
    }
    const uint32_t H = w0->n_head_kv, D = w0->head_dim;
    if (n_head == 0 || n_head % H) return kvm_fail(st, KVM_EINVAL, "%s: %u heads on %u", what, n_head, H);
    if (!std::isfinite(scale)) return kvm_fail(st, KVM_EINVAL, "%s: scale %g", what, (double)scale);
    if (total * (n_head / H) > (1u << 24)) return kvm_fail(st, KVM_ERANGE, "%s: %llu tokens", what, (unsigned long long)total);
    if (H > 65535) return kvm_fail(st, KVM_ERANGE, "%s: %u kv heads", what, H);
    if (total == 0) return KVM_OK;
    if (!q || !q_pos || !out) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    fs_args a{};
    a.H = H;
    a.G = n_head / H;
    a.n_head = n_head;
    a.n_rows = (uint32_t)total * a.G;
    a.q = q;
    a.q_type = q_type;
    a.q_pos = q_pos;
    a.out = out;
    a.out_type = out_type;
    a.q_sign = scale < 0.0f ? -1.0f : scale > 0.0f ? 1.0f : 0.0f;
    a.c = scale != 0.0f ? fabsf(scale) * 1.4426950408889634f : 1.0f;
    uint32_t units = 0;
    const bool quant = kvm_k_quant(w0->k_type);
    const uint32_t n_wg = (st ? st->n_cu : 256u) * fs_resident(D, quant);
    const int rc = fs_shape(st, what, prefix, windows, n_tokens, n_lanes, n_wg, &a, &units);
    if (rc) return rc;
    if (!st) return KVM_EINVAL;
    const uint64_t slots = a.n_seg ? (1ull << a.log_p) + units : 0;
    const size_t bytes_o = (size_t)slots * 32 * D * 4, bytes = bytes_o + (size_t)slots * 32 * 8;
    KVM_HIP(st, hipSetDevice(st->device));
    if (slots) {
        void *ws = nullptr;
        if (const int bad = kvm_shared_workspace(st, what, bytes, &ws)) return bad;
        a.ws_o = (float *)ws;
        a.ws_ml = (float *)((uint8_t *)a.ws_o + bytes_o);
    }
    auto go = [&](auto d) {
        constexpr int DD = decltype(d)::value;
        if (a.n_seg) {
            if (quant) hipLaunchKernelGGL((k_fs_attn<DD, true>), dim3(1u << a.log_p), dim3(256), 0, st->stream, a);
            else hipLaunchKernelGGL((k_fs_attn<DD, false>), dim3(1u << a.log_p), dim3(256), 0, st->stream, a);
        }
        hipLaunchKernelGGL((k_fs_join<DD, 4>), dim3(kvm_cdiv(a.n_rows, 32), DD / 8, H), dim3(256), 0, st->stream, a);
    };
    if (D == 256) go(std::integral_constant<int, 256>{});
    else go(std::integral_constant<int, 128>{});
    KVM_LAUNCH_CHECK(st, what);
    return KVM_OK;
}
