// kvm_append.hip -- what a layer does with its new tokens before it attends: norms of
// the queries and keys of each head with the position rotation in the same pass
// (kvm_qk_norm_rope), and the keys and values into the cells of their windows
// (kvm_window_append).
//
// A row is one head of one token.  With x its D values,
//   r = 1 / sqrt(mean x_d^2 + eps), formed in 64 bits and rounded once,
//   y_d = (x_d r) w_d,
//   pairs (i, i + n_rot / 2), angle a = fl32(pos theta_i): y_i' = y_i cos a - y_j sin a,
//   y_j' = y_i sin a + y_j cos a,
//   the normalised Walsh-Hadamard transform of chunks of nrot dims: pre-scaled by
//   1 / sqrt(nrot), butterflies h = 1, 2, ..
// each operation one fp32 rounding, cos a and sin a the roundings of the 64-bit values.
// The sum of squares does not depend on the order of its terms then (a 64-bit sum's
// order changes r in one row of some 1e8), the angles are those of the stage-in's table,
// and a key row equals the stage-in's for the same values and position.
#include "kvm_internal.h"

#include <cmath>
#include <type_traits>

#define KVM_APPEND_RUNS 40u      // runs of one launch: their descriptors are kernel arguments

typedef __bf16 kvm_bf16x4 __attribute__((ext_vector_type(4)));

// ---- device: angles -----------------------------------------------------------
// cos and sin of an fp32 angle to within an ulp of 64 bits: a - k pi/2 with pi/2 in two
// doubles (one rounding each, by fma), then the Taylor series, whose first terms left
// out are below 2^-57 for |r| <= pi/4.
__device__ inline float2 cos_sin(float angle) {
    const double a = (double)angle, k = rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-k, 1.57079632679489661923, a);
    r = __builtin_fma(-k, 6.123233995736766036e-17, r);
    const double z = r * r;
    double c = 1.0 / 20922789888000.0, s = -1.0 / 1307674368000.0;      // 1 / 16!, -1 / 15!
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, r, r);
    const int quarter = (int)(k - 4.0 * floor(k * 0.25));
    const double cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    return make_float2((float)(quarter == 1 || quarter == 2 ? -cc : cc), (float)(quarter >= 2 ? -ss : ss));
}

struct head_args {
    uint32_t D, n_half;          // values of a row; rotated pairs, 0 = no rotation
    int32_t nrot;                // Walsh-Hadamard width, 0 = none
    int32_t norm;                // 0: rows are taken as they are
    float hscale, eps;
    double inv_D;
    float theta[128];
};

struct head_src {
    const uint8_t *data;
    int type;
    size_t nb0, nb1, nb2;        // bytes from a dim, a head, a token to the next
    const float *weight;         // [D] or null
};

// ---- device: rows ---------------------------------------------------------------
// LPR lanes hold a row, 4 consecutive dims each, a wave 64 / LPR rows at a time and NI
// times that in all, loaded before the first is used.
template <typename T>
__device__ __forceinline__ T ld_any(const void *p) {
    T x;
    __builtin_memcpy(&x, p, sizeof(T));
    return x;
}
__device__ __forceinline__ uint32_t elem_size(int type) { return type == KVM_TYPE_F32 ? 4u : 2u; }
__device__ __forceinline__ float from16(int type, uint32_t u) { return type == KVM_TYPE_BF16 ? kvm_bf2f((uint16_t)u) : kvm_h2f((uint16_t)u); }
// 4 dims of a row at p, any strides and type
__device__ __forceinline__ void load4(const head_src &s, const uint8_t *p, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = s.type == KVM_TYPE_F32 ? ld_any<float>(p + i * s.nb0) : from16(s.type, ld_any<uint16_t>(p + i * s.nb0));
}

#define DPP_QUAD(a, b, c, d) ((a) | (b) << 2 | (c) << 4 | (d) << 6)
// A 64-bit value of another lane, as a DPP move of its halves.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// x of lane l ^ O (O = 16 and 32: the swap leaves the lower rows' own value and the upper
// rows' partner in one result, the others in the other)
template <int O>
__device__ __forceinline__ float xor_f32(float x) {
    if constexpr (O == 1) return dpp_f32<DPP_QUAD(1, 0, 3, 2)>(x);
    else if constexpr (O == 2) return dpp_f32<DPP_QUAD(2, 3, 0, 1)>(x);
    else if constexpr (O == 4) return dpp_f32<DPP_QUAD(3, 2, 1, 0)>(dpp_f32<0x141>(x));      // row_half_mirror: l ^ 7
    else if constexpr (O == 8) return dpp_f32<0x128>(x);                                       // row_ror:8
    else {
        const uint32_t u = __float_as_uint(x);
        const auto r = O == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return __uint_as_float(threadIdx.x & O ? r[0] : r[1]);
    }
}
// x of the even and of the odd row of 16 lanes (or half of 32) of a pair, added: the same in both.
template <int N>
__device__ __forceinline__ double add_rows_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
    const auto a = N == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false) : __builtin_amdgcn_permlane32_swap(l, l, false, false);
    const auto b = N == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false) : __builtin_amdgcn_permlane32_swap(h, h, false, false);
    return __builtin_bit_cast(double, (uint64_t)b[0] << 32 | a[0]) + __builtin_bit_cast(double, (uint64_t)b[1] << 32 | a[1]);
}
// 1 / sqrt(m) to within some ulps of 64 bits: two Newton steps from the hardware's
// estimate (m is at least the square of the smallest fp32, or 0, infinite or no number).
__device__ __forceinline__ double recip_sqrt(double m) {
    double y = __builtin_amdgcn_rsq(m);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double e = __builtin_fma(-m * y, y, 1.0);
        y = __builtin_fma(0.5 * y, e, y);
    }
    return m > 0.0 && m < (double)INFINITY ? y : 1.0 / sqrt(m);
}

template <int LPR, int NI>
struct head_rows {
    static constexpr int RPW = 64 / LPR, ROWS = 4 * RPW * NI;    // rows of a wave at a time, of a workgroup
    float x[NI][4];
    uint32_t t[NI], h[NI];       // token of the block, head
    bool live[NI];

    // The rows of tokens [t0, t0 + nt) and heads [h0, h0 + nh), nt nh <= ROWS; heads from
    // `split` on are the second tensor's.
    __device__ __forceinline__ void load(const head_args &a, const head_src &s, const head_src &s2, uint32_t split, uint32_t t0,
                                         uint32_t nt, uint32_t h0, uint32_t nh) {
        const uint32_t l = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d0 = 4 * (l % LPR);
        const uint8_t *p[NI];            // the rows (one a wave: in scalar registers)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            // (a row past the last is the unit's first, its dims past D are dim 0: loaded, not used)
            const uint32_t r = (i * 4 + w) * RPW + (RPW > 1 ? l / LPR : 0u);
            live[i] = r < nt * nh;
            t[i] = live[i] ? r / nh : 0u;
            h[i] = h0 + (live[i] ? r - t[i] * nh : 0u);
            const size_t tok = t0 + t[i];
            p[i] = h[i] < split ? s.data + tok * s.nb2 + (size_t)h[i] * s.nb1 : s2.data + tok * s2.nb2 + (size_t)(h[i] - split) * s2.nb1;
        }
        // Rows of packed dims are loaded first and converted after: a conversion waits for
        // its load, one row's after the other.
        const uint32_t es = elem_size(s.type), d = d0 < a.D ? d0 : 0u;
        const bool packed = s.nb0 == es && s2.nb0 == es && elem_size(s2.type) == es;
        if (packed && es == 4) {
            kvm_f32x4 v[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) v[i] = ld_any<kvm_f32x4>(p[i] + 4 * d);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = v[i][j];
        } else if (packed) {
            kvm_u32x2 v[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) v[i] = ld_any<kvm_u32x2>(p[i] + 2 * d);
            if (s.type == KVM_TYPE_BF16 && s2.type == KVM_TYPE_BF16) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = __uint_as_float(j & 1 ? v[i][j >> 1] & 0xffff0000u : v[i][j >> 1] << 16);
            } else {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = from16(h[i] < split ? s.type : s2.type, j & 1 ? v[i][j >> 1] >> 16 : v[i][j >> 1] & 0xffffu);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const head_src &q = h[i] < split ? s : s2;
                load4(q, p[i] + d * q.nb0, x[i]);
            }
        }
        if (d0 >= a.D) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = 0.0f;
        }
    }

    // norm, rotation, transform; cs: (cos, sin) of [token of the block][pair], nt tokens
    __device__ __forceinline__ void turn(const head_args &a, const float *weight, const float *weight2, uint32_t split,
                                         const float2 *cs, uint32_t nt) {
        const uint32_t l = threadIdx.x & 63u, d0 = 4 * (l % LPR);
        if (a.norm) {
            const kvm_f32x4 ones = {1.0f, 1.0f, 1.0f, 1.0f};
            const kvm_f32x4 w = weight && d0 < a.D ? ld_any<kvm_f32x4>(weight + d0) : ones;
            const kvm_f32x4 w2 = weight2 && d0 < a.D ? ld_any<kvm_f32x4>(weight2 + d0) : ones;
            double sum[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                sum[i] = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i] = __builtin_fma((double)x[i][j], (double)x[i][j], sum[i]);
            }
            // Over the lanes of a row.  With four rows, lane l keeps row l % 4 after two
            // exchanges, so that one root serves all four.
            static_assert(NI == 1 || NI == 4, "rows of a wave");
            double v;
            if constexpr (NI == 4) {
                const bool o1 = l & 1u, o2 = l & 2u;
                const double a0 = (o1 ? sum[1] : sum[0]) + dpp_f64<DPP_QUAD(1, 0, 3, 2)>(o1 ? sum[0] : sum[1]);
                const double a1 = (o1 ? sum[3] : sum[2]) + dpp_f64<DPP_QUAD(1, 0, 3, 2)>(o1 ? sum[2] : sum[3]);
                v = (o2 ? a1 : a0) + dpp_f64<DPP_QUAD(2, 3, 0, 1)>(o2 ? a0 : a1);
            } else {
                v = sum[0] + dpp_f64<DPP_QUAD(1, 0, 3, 2)>(sum[0]);
                v += dpp_f64<DPP_QUAD(2, 3, 0, 1)>(v);
            }
            v += dpp_f64<0x124>(v);                      // row_ror:4
            v += dpp_f64<0x128>(v);                      // row_ror:8
            if constexpr (LPR >= 32) v = add_rows_f64<16>(v);
            if constexpr (LPR >= 64) v = add_rows_f64<32>(v);
            const float root = (float)recip_sqrt(__builtin_fma(v, a.inv_D, (double)a.eps));
            auto scale = [&](auto row) {
                constexpr int i = decltype(row)::value;
                const float r = NI == 1 ? root : __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(root), DPP_QUAD(i, i, i, i), 0xf, 0xf, true));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = kvm_fmul(kvm_fmul(x[i][j], r), h[i] < split ? w[j] : w2[j]);
            };
            scale(std::integral_constant<int, 0>{});
            if constexpr (NI == 4) {
                scale(std::integral_constant<int, 1>{});
                scale(std::integral_constant<int, 2>{});
                scale(std::integral_constant<int, 3>{});
            }
        }
        if (d0 < 2 * a.n_half) {
            // the partner's lane, one that turns too: n_half is a multiple of 4
            const bool lo = d0 < a.n_half;
            const uint32_t pl = a.n_half / 4, p = (lo ? l + pl : l - pl) << 2, ci = lo ? d0 : d0 - a.n_half;
            const uint32_t sm = lo ? 0x80000000u : 0u;
            float y[NI][4];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) y[i][j] = __int_as_float(__builtin_amdgcn_ds_bpermute((int)p, __float_as_int(x[i][j])));
            float c[4], sn[4];
            auto angles = [&](uint32_t token) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = cs[token * a.n_half + ci + j];
                    c[j] = v.x;
                    sn[j] = __uint_as_float(__float_as_uint(v.y) ^ sm);
                }
            };
            auto rotate = [&](int i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = kvm_fadd(kvm_fmul(x[i][j], c[j]), kvm_fmul(y[i][j], sn[j]));
            };
            if (nt == 1) {                       // one token's rows turn alike
                angles(0);
#pragma unroll
                for (int i = 0; i < NI; ++i) rotate(i);
            } else {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    angles(t[i]);
                    rotate(i);
                }
            }
        }
        if (a.nrot) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = kvm_fmul(x[i][j], a.hscale);
                x[i][0] = kvm_fadd(y[0], y[1]);
                x[i][1] = kvm_fsub(y[0], y[1]);
                x[i][2] = kvm_fadd(y[2], y[3]);
                x[i][3] = kvm_fsub(y[2], y[3]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float u = x[i][j], v = x[i][j + 2];
                    x[i][j] = kvm_fadd(u, v);
                    x[i][j + 2] = kvm_fsub(u, v);
                }
            }
            auto stage = [&](auto lanes) {
                constexpr int O = decltype(lanes)::value;
                const float sg = l & O ? -1.0f : 1.0f;           // the lane above takes other - own
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = __builtin_fmaf(x[i][j], sg, xor_f32<O>(x[i][j]));
            };
            stage(std::integral_constant<int, 1>{});             // (chunks of 64 dims at least)
            stage(std::integral_constant<int, 2>{});
            stage(std::integral_constant<int, 4>{});
            stage(std::integral_constant<int, 8>{});
            if constexpr (LPR >= 32)
                if (a.nrot > 64) stage(std::integral_constant<int, 16>{});
            if constexpr (LPR >= 64)
                if (a.nrot > 128) stage(std::integral_constant<int, 32>{});
        }
    }

    // rows out [token][head][D] of `type`, the two tensors' heads (split and the rest of n_head) apart
    __device__ __forceinline__ void store(const head_args &a, uint8_t *out, uint8_t *out2, uint32_t split, uint32_t n_head, int type,
                                          uint32_t t0) const {
        const uint32_t d0 = 4 * ((threadIdx.x & 63u) % LPR);
        if (d0 >= a.D) return;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if (!live[i]) continue;
            const bool first = h[i] < split;
            const size_t row = (size_t)(t0 + t[i]) * (first ? split : n_head - split) + (first ? h[i] : h[i] - split);
            uint8_t *o = (first ? out : out2) + row * a.D * elem_size(type);
            const kvm_f32x4 v = {x[i][0], x[i][1], x[i][2], x[i][3]};
            if (type == KVM_TYPE_F32) {
                __builtin_memcpy(o + 4 * d0, &v, 16);
            } else if (type == KVM_TYPE_BF16) {
                const kvm_bf16x4 u = __builtin_convertvector(v, kvm_bf16x4);
                __builtin_memcpy(o + 2 * d0, &u, 8);
            } else {
                uint32_t u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = kvm_f2h(v[j]);
                const kvm_u32x2 y = {u[0] | u[1] << 16, u[2] | u[3] << 16};
                __builtin_memcpy(o + 2 * d0, &y, 8);
            }
        }
    }
};

// (cos, sin) of the positions of tokens [t0, t0 + nt)
__device__ __forceinline__ void fill_cs(const head_args &a, const int32_t *pos, uint32_t t0, uint32_t nt, float2 *cs) {
    if (!a.n_half) return;
    for (uint32_t i = threadIdx.x; i < nt * a.n_half; i += 256) {
        const uint32_t t = i / a.n_half, j = i - t * a.n_half;
        cs[i] = cos_sin(kvm_fmul((float)pos[t0 + t], a.theta[j]));
    }
    __syncthreads();
}

// The rows of a launch's queries (and keys), in units of tt tokens x hb heads.
struct rope_args {
    head_src q, k;
    const int32_t *pos;
    uint8_t *q_out, *k_out;
    int type;
    uint32_t n_tokens, n_head, split;    // heads of both, of the queries
    uint32_t tt, hb, units;
};

template <int LPR, int NI>
__device__ __forceinline__ void norm_rope_unit(const head_args &a, const rope_args &u, uint32_t unit, float2 *cs) {
    const uint32_t nhb = (u.n_head + u.hb - 1) / u.hb, t0 = unit / nhb * u.tt, h0 = unit % nhb * u.hb;
    const uint32_t nt = min(u.tt, u.n_tokens - t0), nh = min(u.hb, u.n_head - h0);
    head_rows<LPR, NI> r;
    r.load(a, u.q, u.k, u.split, t0, nt, h0, nh);
    fill_cs(a, u.pos, t0, nt, cs);
    r.turn(a, u.q.weight, u.k.weight, u.split, cs, nt);
    r.store(a, u.q_out, u.k_out, u.split, u.n_head, u.type, t0);
}

struct norm_rope_args {
    head_args a;
    rope_args u;
};

// What bounds it: the memory for many rows (2,048 tokens of 28 x 256 in bf16: 16.1 us for 58.7
// MB, 3.7 TB/s), one round trip and the launch for few (a token: 4.6 us).
template <int LPR, int NI>
__global__ void __launch_bounds__(256) k_norm_rope(norm_rope_args g) {
    __shared__ float2 s_cs[512 * NI];    // ROWS tokens of 2 LPR pairs at most
    norm_rope_unit<LPR, NI>(g.a, g.u, blockIdx.x, s_cs);
}

// ---- device: keys and values into a window ---------------------------------------
// A run: tokens tok0 .. tok0 + n - 1 of the call into cells cell0 .. of a window.  No two
// runs of a launch touch the same 8-cell group or slot of a window: what is read and
// written back (the words of 8 cells' nibbles, the slots' counts) has one owner.
struct run_args {
    uint8_t *k, *v;
    int32_t *cell_pos;
    uint32_t *shadow_rows, *pending;     // null, or the slots' counts
    uint32_t n_tiles, bt;
    uint32_t cell0, n, tok0;
};

struct append_args {
    head_args a;
    rope_args u;                 // the queries
    head_src k, v;
    const int32_t *pos;
    uint32_t H, n_runs;
    uint32_t tk, hk;             // tokens and heads of a key unit
    uint32_t u0[KVM_APPEND_RUNS];        // first units, ascending
    run_args run[KVM_APPEND_RUNS];
};
static_assert(sizeof(append_args) <= 4096, "kernel arguments");

// One (8-cell group, head) of the values: lane d of the D that share it has dim d of the
// group's tokens, so a word (8 nibbles) or 16 bytes (8 halves) of the tile is a lane's own.
template <int D, bool QUANT>
__device__ __forceinline__ void append_v(const append_args &g, const run_args &r, uint32_t h, uint32_t grp, uint32_t d) {
    const uint32_t c0 = 8 * grp;         // the group's first cell
    const uint8_t *base = g.v.data + (size_t)h * g.v.nb1 + (size_t)d * g.v.nb0;
    const uint8_t *p[8];
    float x[8];
    uint32_t valid = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t i = c0 + j - r.cell0;                     // token of the run (wraps below cell0)
        const bool in = c0 + j >= r.cell0 && i < r.n;
        valid |= (uint32_t)in << j;
        p[j] = base + (size_t)(r.tok0 + (in ? i : c0 + j < r.cell0 ? 0u : r.n - 1)) * g.v.nb2;
    }
    uint8_t *vt = r.v + ((size_t)h * r.n_tiles + c0 / 64) * kvm_vtile_bytes(QUANT ? KVM_TYPE_Q4_0 : KVM_TYPE_F16, D);
    const uint32_t c = c0 % 64;
    uint32_t *const word_at = (uint32_t *)(vt + kvm_vq_word(d, (c & 31u) >> 3, c >> 5));
    uint32_t old = 0;
    if (QUANT && valid != 0xffu) old = *word_at;                 // the other cells' nibbles stay
    if (g.v.type == KVM_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = ld_any<float>(p[j]);
    } else {
        uint16_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = ld_any<uint16_t>(p[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = from16(g.v.type, u[j]);
    }
    if constexpr (!QUANT) {
        uint16_t *dst = (uint16_t *)vt + kvm_vh_idx(c, d);
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = kvm_f2h(x[j]);
        if (valid == 0xffu) {
            *(kvm_u32x4 *)dst = kvm_u32x4{y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (valid >> j & 1u) dst[j] = (uint16_t)y[j];
        }
    } else {
        const uint32_t l = threadIdx.x & 31u;
        uint32_t word = 0, mask = 0;
        uint16_t *sc = (uint16_t *)(vt + kvm_vd_off(D, c, d / 32));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // the block's largest magnitude, with the sign of the first in dim order
            const float ax = fabsf(x[j]);
            float m = fmaxf(ax, xor_f32<1>(ax));
            m = fmaxf(m, xor_f32<2>(m));
            m = fmaxf(m, dpp_f32<0x124>(m));                     // row_ror:4, :8: the row's four quads
            m = fmaxf(m, xor_f32<8>(m));
            m = kvm_max_xor16(m);
            const uint64_t eq = __builtin_amdgcn_ballot_w64(ax == m), neg = __builtin_amdgcn_ballot_w64(x[j] < 0.0f);
            const uint32_t eq32 = (uint32_t)(threadIdx.x & 32u ? eq >> 32 : eq), neg32 = (uint32_t)(threadIdx.x & 32u ? neg >> 32 : neg);
            const bool minus = neg32 & eq32 & (0u - eq32);       // (the lowest set bit)
            const float dsc = m > 0.0f ? kvm_fmul(minus ? -m : m, -0.125f) : -0.0f;
            int n = (int)kvm_fadd(kvm_fmul(x[j], kvm_recip_or0(dsc)), 8.5f);
            n = n > 15 ? 15 : n;
            if (valid >> j & 1u) {
                mask |= 15u << kvm_vq_nib_shift(j);
                word |= (uint32_t)(n & 15) << kvm_vq_nib_shift(j);
                if (l == 0) sc[j] = kvm_f2h(dsc);
            }
        }
        *word_at = word | (old & ~mask);
    }
}

// Key rows, 4 dims a lane: into the tile at cell c.
template <int D, int KT, int NI>
__device__ __forceinline__ void append_k(const head_rows<D / 4, NI> &r, const run_args &run, uint32_t cell) {
    const uint32_t l = threadIdx.x & 63u, d0 = 4 * (l % (D / 4)), b = d0 / 32;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const uint32_t at = cell + r.t[i], c = at % 64;
        uint8_t *kt = run.k + ((size_t)r.h[i] * run.n_tiles + at / 64) * kvm_ktile_bytes(KT, D);
        if constexpr (KT == KVM_TYPE_F16) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = kvm_f2h(r.x[i][j]);
            if (r.live[i]) *(kvm_u32x2 *)((uint16_t *)kt + kvm_kh_idx(D, c, d0)) = kvm_u32x2{y[0] | y[1] << 16, y[2] | y[3] << 16};
        } else {
            // a block's 32 dims are 8 lanes'
            float m = fmaxf(fmaxf(fabsf(r.x[i][0]), fabsf(r.x[i][1])), fmaxf(fabsf(r.x[i][2]), fabsf(r.x[i][3])));
            m = fmaxf(m, xor_f32<1>(m));
            m = fmaxf(m, xor_f32<2>(m));
            m = fmaxf(m, dpp_f32<0x141>(m));                     // row_half_mirror: the other quad
            float d;
            if constexpr (KT == KVM_TYPE_Q8_0) {
                d = kvm_div127(m);
            } else {
                // the sign of the first value of that magnitude in dim order
                uint32_t first = 0xffu;
#pragma unroll
                for (int j = 3; j >= 0; --j)
                    if (fabsf(r.x[i][j]) == m) first = 2 * (4 * (l & 7u) + j) + (__float_as_uint(r.x[i][j]) >> 31);
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) first = min(first, (uint32_t)__shfl_xor((int)first, o, 64));
                d = m > 0.0f ? kvm_fmul(first & 1u ? -m : m, -0.125f) : -0.0f;
            }
            const float id = kvm_recip_or0(d);
            uint32_t qw = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int q;
                if constexpr (KT == KVM_TYPE_Q8_0) {
                    q = kvm_round_away(kvm_fmul(r.x[i][j], id));
                } else {
                    q = (int)kvm_fadd(kvm_fmul(r.x[i][j], id), 8.5f);
                    q = (q > 15 ? 15 : q) - 8;
                }
                qw |= (uint32_t)(uint8_t)(int8_t)q << (8 * j);
            }
            if (!r.live[i]) continue;
            *(uint32_t *)(kt + kvm_kq_off(D, c, d0)) = qw;
            if ((l & 7u) == 0) *(uint16_t *)(kt + kvm_kd_off(D, c, b)) = kvm_f2h(d);
        }
    }
}

// Queries, keys, values and positions are units of one launch: none of them waits for another.
// What bounds it: for many tokens the arithmetic of the rows (norm, transform, quantisation) and
// two round trips (2,047 tokens of 4 x 256 into q8_0 / q4_0: 11.8 us, 11.8 MB; the memory alone
// 2.4), for few the launch and a round trip (a token: 4.4 us).
template <int D, int KT, int NI>
__global__ void __launch_bounds__(256) k_append(append_args g) {
    __shared__ float2 s_cs[512 * NI];
    constexpr bool QUANT = KT != KVM_TYPE_F16;
    uint32_t b = blockIdx.x;
    if (b < g.u.units) return norm_rope_unit<D / 4, NI>(g.a, g.u, b, s_cs);
    b -= g.u.units;
    // The unit's run: the last of those that begin at or before it.  (Every wave looks at
    // all of them at once; one after the other they are a chain of loads.)
    uint32_t ri = 0;
    if (g.n_runs > 1) {
        const uint32_t lane = threadIdx.x & 63u;
        ri = __builtin_amdgcn_readfirstlane(__popcll(__builtin_amdgcn_ballot_w64(lane < g.n_runs && g.u0[lane < g.n_runs ? lane : 0u] <= b)) - 1);
    }
    const run_args &r = g.run[ri];
    b -= g.u0[ri];
    // the run's units: keys, values, then the positions and the slots' counts
    const uint32_t nhb = (g.H + g.hk - 1) / g.hk, nk = (r.n + g.tk - 1) / g.tk * nhb;
    if (b < nk) {
        const uint32_t i0 = b / nhb * g.tk, nt = min(g.tk, r.n - i0), h0 = b % nhb * g.hk;
        head_rows<D / 4, NI> rows;
        rows.load(g.a, g.k, g.k, g.H, r.tok0 + i0, nt, h0, min(g.hk, g.H - h0));
        fill_cs(g.a, g.pos, r.tok0 + i0, nt, s_cs);
        rows.turn(g.a, g.k.weight, nullptr, g.H, s_cs, nt);
        append_k<D, KT, NI>(rows, r, r.cell0 + i0);
        return;
    }
    b -= nk;
    // (8-cell group, head) pairs, 256 / D of them a unit
    const uint32_t g0 = r.cell0 / 8, pairs = ((r.cell0 + r.n - 1) / 8 - g0 + 1) * g.H, nv = (pairs + 256 / D - 1) / (256 / D);
    if (b < nv) {
        const uint32_t p = b * (256 / D) + __builtin_amdgcn_readfirstlane(threadIdx.x / D);
        if (p < pairs) append_v<D, QUANT>(g, r, p % g.H, g0 + p / g.H, threadIdx.x % D);
        return;
    }
    for (uint32_t i = threadIdx.x; i < r.n; i += 256) r.cell_pos[r.cell0 + i] = g.pos[r.tok0 + i];
    const uint32_t end = r.cell0 + r.n;
    for (uint32_t slot = r.cell0 / r.bt + threadIdx.x; slot * r.bt < end; slot += 256) {
        if (r.shadow_rows) r.shadow_rows[slot] = 0u;
        if (r.pending) {
            const uint32_t rows = min((slot + 1) * r.bt, end) - slot * r.bt;
            r.pending[slot] = max(r.pending[slot], rows);
        }
    }
}

// ---- host -----------------------------------------------------------------------
static int head_args_of(kvm_state *st, const char *what, uint32_t D, float eps, const kvm_rope_params *rope, int nrot, head_args *a) {
    if (std::isnan(eps)) return kvm_fail(st, KVM_EINVAL, "%s: eps is not a number", what);
    a->D = D;
    a->inv_D = 1.0 / (double)D;
    a->norm = eps >= 0.0f;
    a->eps = eps;
    if (!rope) return KVM_OK;
    if (rope->n_rot % 8 || rope->n_rot > D)
        return kvm_fail(st, KVM_EUNSUPPORTED, "%s: n_rot %u (needs a multiple of 8 <= head_dim)", what, rope->n_rot);
    if (rope->n_rot && !(rope->freq_base > 0.0f))
        return kvm_fail(st, KVM_EINVAL, "%s: freq_base %g", what, (double)rope->freq_base);
    if (!kvm_hadamard_ok(nrot, D))
        return kvm_fail(st, KVM_EUNSUPPORTED, "%s: hadamard width %d", what, nrot);
    a->n_half = rope->n_rot / 2;
    a->nrot = nrot;
    a->hscale = nrot ? 1.0f / sqrtf((float)nrot) : 1.0f;
    for (uint32_t i = 0; i < a->n_half; ++i)     // kvm_rope_theta's
        a->theta[i] = powf(rope->freq_base, -2.0f * (float)i / (float)rope->n_rot) * rope->freq_scale;
    return KVM_OK;
}

// A view as rows of D dims: [tokens][heads][D], or with the heads of a token packed in
// one or several longer rows.
static int head_src_of(kvm_state *st, const char *what, const kvm_view *v, uint32_t D, uint32_t n_head, const float *weight, head_src *s) {
    kvm_view some = *v;
    if (v->ne2 == 0 && !v->data) some.data = &some;     // no tokens: no memory either
    const int rc = view_check(st, &some, n_head * D, what);
    if (rc) return rc;
    if (v->ne2 > 0x7fffffff) return kvm_fail(st, KVM_ERANGE, "%s: %lld tokens", what, (long long)v->ne2);
    *s = head_src{(const uint8_t *)v->data, v->type, v->nb0, v->nb1, v->nb2, weight};
    if (v->ne0 == (int64_t)D) return KVM_OK;
    if (v->ne0 % D == 0 && (v->ne1 == 1 || v->nb1 == (size_t)v->ne0 * v->nb0)) {
        s->nb1 = D * v->nb0;
        return KVM_OK;
    }
    return kvm_fail(st, KVM_EUNSUPPORTED, "%s: view rows of %lld values, heads of %u", what, (long long)v->ne0, D);
}

// Rows out: the output may be the rows' own memory, packed and of the same type (a row is
// read before it is written, by the same lanes), but overlap no input otherwise.
static bool overlaps(const void *out, size_t bytes, const kvm_view *v) {
    if (!v || v->ne2 == 0) return false;
    const size_t es = v->type == KVM_TYPE_F32 ? 4 : 2;
    const uintptr_t a = (uintptr_t)out, b = (uintptr_t)v->data;
    const uintptr_t e = b + (size_t)(v->ne2 - 1) * v->nb2 + (size_t)(v->ne1 - 1) * v->nb1 + (size_t)(v->ne0 - 1) * v->nb0 + es;
    return a < e && b < a + bytes;
}
static bool in_place(const void *out, int type, const head_src &s, uint32_t D, uint32_t n_head) {
    const size_t es = type == KVM_TYPE_F32 ? 4 : 2;
    return out == s.data && type == s.type && s.nb0 == es && s.nb1 == D * es && s.nb2 == (size_t)n_head * D * es;
}

static bool float_type(int t) { return t == KVM_TYPE_F32 || t == KVM_TYPE_F16 || t == KVM_TYPE_BF16; }

// Units of at most `rows` rows: the heads in equal parts, and as many tokens as fit.
static void units_of(uint32_t n_tokens, uint32_t n_head, uint32_t rows, uint32_t *tt, uint32_t *hb, uint32_t *units) {
    *hb = kvm_cdiv(n_head, kvm_cdiv(n_head, rows));
    *tt = rows / *hb;
    *units = kvm_cdiv(n_tokens, *tt) * kvm_cdiv(n_head, *hb);
}

// Rows of a wave: one, or four with one root for all.  One hides more latency while the
// chip is not full: us with one and four, keys and values of n tokens of 4 x 256 into a
// quantised window, 512: 6.6 and 7.2, 1,024: 8.8 and 7.7, 2,048: 12.3 and 11.2; norms and
// rotation of 28 x 256, 128: 3.8 and 4.8, 256: 6.2 and 5.7, 2,048: 24.6 and 16.9; of 10 x
// 128, 1,024: 5.9 and 6.1, 2,048: 8.4 and 7.4.
template <typename F>
static void by_ni(uint64_t n_rows, uint32_t rows1, uint32_t n_cu, F &&f) {
    if (n_rows < 4ull * n_cu * rows1) f(std::integral_constant<int, 1>{});
    else f(std::integral_constant<int, 4>{});
}

extern "C" int kvm_qk_norm_rope(kvm_state *st, const kvm_view *q, const kvm_view *k, const float *q_weight,
                                const float *k_weight, float eps, const kvm_rope_params *rope, const int32_t *pos,
                                int out_type, void *q_out, void *k_out) {
    const char *what = "qk_norm_rope";
    if (!q && !k) return kvm_fail(st, KVM_EINVAL, "%s: no queries and no keys", what);
    if (!float_type(out_type)) return kvm_fail(st, KVM_EUNSUPPORTED, "%s: output type %d", what, out_type);
    const kvm_view *one = q ? q : k;
    if (one->ne0 <= 0 || one->ne0 % 8 || one->ne0 > 256) return kvm_fail(st, KVM_EUNSUPPORTED, "%s: head_dim %lld (needs a multiple of 8 <= 256)", what, (long long)one->ne0);
    if (q && k && (q->ne0 != k->ne0 || q->ne2 != k->ne2)) return kvm_fail(st, KVM_EINVAL, "%s: queries and keys of different head_dim or tokens", what);
    for (const kvm_view *v : {q, k})
        if (v && (v->ne1 <= 0 || v->ne1 > (1 << 20))) return kvm_fail(st, KVM_ERANGE, "%s: %lld heads", what, (long long)v->ne1);
    if (rope && rope->hadamard_nrot < 0) return kvm_fail(st, KVM_EINVAL, "%s: hadamard width %d (there is no window to take it from)", what, rope->hadamard_nrot);
    norm_rope_args g{};
    const uint32_t D = (uint32_t)one->ne0;
    int rc = head_args_of(st, what, D, eps, rope, rope ? rope->hadamard_nrot : 0, &g.a);
    if (rc) return rc;
    const size_t es = out_type == KVM_TYPE_F32 ? 4 : 2;
    uint32_t Hq = 0, Hk = 0;
    if (q) {
        Hq = (uint32_t)q->ne1;
        if ((rc = head_src_of(st, what, q, D, Hq, q_weight, &g.u.q))) return rc;
    }
    if (k) {
        Hk = (uint32_t)k->ne1;
        if ((rc = head_src_of(st, what, k, D, Hk, k_weight, &g.u.k))) return rc;
    }
    const uint32_t n = (uint32_t)one->ne2;
    const uint64_t n_rows = (uint64_t)n * (Hq + Hk);
    if (n == 0) return KVM_OK;
    if (n_rows > (1u << 30)) return kvm_fail(st, KVM_ERANGE, "%s: %u tokens", what, n);
    if ((q && !q_out) || (k && !k_out) || (g.a.n_half && !pos)) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    const size_t bq = (size_t)n * Hq * D * es, bk = (size_t)n * Hk * D * es;
    if ((q && ((overlaps(q_out, bq, q) && !in_place(q_out, out_type, g.u.q, D, Hq)) || overlaps(q_out, bq, k))) ||
        (k && ((overlaps(k_out, bk, k) && !in_place(k_out, out_type, g.u.k, D, Hk)) || overlaps(k_out, bk, q))) ||
        (q && k && (uint8_t *)q_out < (uint8_t *)k_out + bk && (uint8_t *)k_out < (uint8_t *)q_out + bq && bq))
        return kvm_fail(st, KVM_EINVAL, "%s: an output overlaps an input or the other output", what);
    if (!st) return KVM_EINVAL;
    if (!q) g.u.q = g.u.k;       // (no head is read from it)
    if (!k) g.u.k = g.u.q;
    g.u.pos = pos;
    g.u.q_out = (uint8_t *)q_out;
    g.u.k_out = (uint8_t *)k_out;
    g.u.type = out_type;
    g.u.n_tokens = n;
    g.u.n_head = Hq + Hk;
    g.u.split = Hq;
    KVM_HIP(st, hipSetDevice(st->device));
    auto go = [&](auto lpr) {
        constexpr int LPR = decltype(lpr)::value;
        by_ni(n_rows, 4 * (64 / LPR), st->n_cu, [&](auto ni) {
            constexpr int NI = decltype(ni)::value;
            units_of(n, Hq + Hk, head_rows<LPR, NI>::ROWS, &g.u.tt, &g.u.hb, &g.u.units);
            hipLaunchKernelGGL((k_norm_rope<LPR, NI>), dim3(g.u.units), dim3(256), 0, st->stream, g);
        });
    };
    if (D > 128) go(std::integral_constant<int, 64>{});
    else if (D > 64) go(std::integral_constant<int, 32>{});
    else go(std::integral_constant<int, 16>{});
    KVM_LAUNCH_CHECK(st, what);
    return KVM_OK;
}

extern "C" int kvm_window_append(kvm_state *st, const kvm_window *const *windows, const uint32_t *cell0,
                                 const uint32_t *n_tokens, uint32_t n_runs, const kvm_view *k, const kvm_view *v,
                                 const float *k_weight, float eps, const kvm_rope_params *rope, const int32_t *pos,
                                 const kvm_view *q, const float *q_weight, int q_out_type, void *q_out) {
    const char *what = "window_append";
    if (n_runs == 0) {
        for (const kvm_view *x : {k, v, q})
            if (x && x->ne2 != 0) return kvm_fail(st, KVM_EINVAL, "%s: no runs, views of %lld tokens", what, (long long)x->ne2);
        return KVM_OK;
    }
    if (!windows || !cell0 || !n_tokens || !k || !v) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    if (q && !float_type(q_out_type)) return kvm_fail(st, KVM_EUNSUPPORTED, "%s: output type %d", what, q_out_type);
    uint64_t total = 0;
    for (uint32_t i = 0; i < n_runs; ++i) {
        const kvm_window *w = windows[i], *w0 = windows[0];
        const int rc = kvm_window_check(w);
        if (rc) return kvm_fail(st, rc, "%s: run %u: bad window", what, i);
        if (w->n_head_kv != w0->n_head_kv || w->head_dim != w0->head_dim || w->k_type != w0->k_type || w->v_type != w0->v_type)
            return kvm_fail(st, KVM_EUNSUPPORTED, "%s: run %u: windows of different heads or types", what, i);
        if ((uint64_t)cell0[i] + n_tokens[i] > w->n_cells) return kvm_fail(st, KVM_ERANGE, "%s: run %u: cells past the window", what, i);
        total += n_tokens[i];
    }
    const kvm_window *w0 = windows[0];
    const uint32_t D = w0->head_dim, H = w0->n_head_kv;
    append_args g{};
    int rc = head_args_of(st, what, D, eps, rope, rope ? kvm_hadamard_width(w0, rope->hadamard_nrot) : 0, &g.a);
    if (rc) return rc;
    if ((rc = head_src_of(st, what, k, D, H, k_weight, &g.k)) || (rc = head_src_of(st, what, v, D, H, nullptr, &g.v))) return rc;
    uint32_t Hq = 0;
    if (q) {
        if (q->ne0 <= 0 || q->ne1 <= 0 || (uint64_t)q->ne0 * (uint64_t)q->ne1 % D || (uint64_t)q->ne0 * (uint64_t)q->ne1 > (1u << 28))
            return kvm_fail(st, KVM_EINVAL, "%s: queries of %lld x %lld values, heads of %u", what, (long long)q->ne0, (long long)q->ne1, D);
        Hq = (uint32_t)((uint64_t)q->ne0 * (uint64_t)q->ne1 / D);
        if ((rc = head_src_of(st, what, q, D, Hq, q_weight, &g.u.q))) return rc;
    }
    if ((uint64_t)k->ne2 != total || (uint64_t)v->ne2 != total || (q && (uint64_t)q->ne2 != total))
        return kvm_fail(st, KVM_EINVAL, "%s: runs of %llu tokens, keys of %lld, values of %lld", what, (unsigned long long)total, (long long)k->ne2, (long long)v->ne2);
    if (total * (H + Hq) > (1u << 30)) return kvm_fail(st, KVM_ERANGE, "%s: %llu tokens", what, (unsigned long long)total);
    if (total == 0) return KVM_OK;
    if (!pos || (q && !q_out)) return kvm_fail(st, KVM_EINVAL, "%s: null argument", what);
    if (q) {
        const size_t bytes = total * Hq * D * (q_out_type == KVM_TYPE_F32 ? 4 : 2);
        if ((overlaps(q_out, bytes, q) && !in_place(q_out, q_out_type, g.u.q, D, Hq)) || overlaps(q_out, bytes, k) || overlaps(q_out, bytes, v))
            return kvm_fail(st, KVM_EINVAL, "%s: the query output overlaps an input", what);
    }
    if (!st) return KVM_EINVAL;
    g.pos = g.u.pos = pos;
    g.u.q_out = (uint8_t *)q_out;
    g.u.type = q_out_type;
    g.u.n_tokens = (uint32_t)total;
    g.u.n_head = g.u.split = Hq;
    g.u.k = g.u.q;
    g.H = H;
    KVM_HIP(st, hipSetDevice(st->device));

    // Launches of runs that share no 8-cell group and no slot; the first takes the queries.
    uint32_t tok = 0;
    auto shares = [&](uint32_t i, uint32_t j) {
        const kvm_window *a = windows[i], *b = windows[j];
        if (a->k != b->k && a->v != b->v && a->cell_pos != b->cell_pos) return false;
        const uint32_t s = a->block_tokens % 8 ? 1u : a->block_tokens, m = s > 8 && (a->pending_rows || a->shadow_rows) ? s : 8u;
        if (s == 1u) return true;        // (slots that cut the groups)
        return cell0[i] / m <= (cell0[j] + n_tokens[j] - 1) / m && cell0[j] / m <= (cell0[i] + n_tokens[i] - 1) / m;
    };
    by_ni(total * (H + Hq), 4 * (64 / (D / 4)), st->n_cu, [&](auto ni) {
        constexpr int NI = decltype(ni)::value;
        const uint32_t rows = 4 * (256 / D) * NI;
        if (q) units_of((uint32_t)total, Hq, rows, &g.u.tt, &g.u.hb, &g.u.units);
        uint32_t unused;
        units_of((uint32_t)total, H, rows, &g.tk, &g.hk, &unused);
        for (uint32_t i = 0; i < n_runs;) {
            uint32_t first = i, units = 0;
            g.n_runs = 0;
            for (; i < n_runs && g.n_runs < KVM_APPEND_RUNS; ++i) {
                if (!n_tokens[i]) continue;
                bool clash = false;
                for (uint32_t j = first; j < i && !clash; ++j) clash = n_tokens[j] && shares(i, j);
                if (clash) break;
                const kvm_window *w = windows[i];
                g.u0[g.n_runs] = units;
                g.run[g.n_runs++] = run_args{(uint8_t *)w->k, (uint8_t *)w->v, w->cell_pos, w->shadow_rows, w->pending_rows,
                             w->n_cells / KVM_TILE_CELLS, w->block_tokens, cell0[i], n_tokens[i], tok};
                const uint32_t pairs = ((cell0[i] + n_tokens[i] - 1) / 8 - cell0[i] / 8 + 1) * H;
                units += kvm_cdiv(n_tokens[i], g.tk) * kvm_cdiv(H, g.hk) + kvm_cdiv(pairs, 256 / D) + 1;
                tok += n_tokens[i];
            }
            if (!g.n_runs) break;
            auto go = [&](auto d, auto kt) {
                hipLaunchKernelGGL((k_append<decltype(d)::value, decltype(kt)::value, NI>), dim3(g.u.units + units), dim3(256), 0, st->stream, g);
            };
            auto go_d = [&](auto d) {
                if (w0->k_type == KVM_TYPE_Q8_0) go(d, std::integral_constant<int, KVM_TYPE_Q8_0>{});
                else if (w0->k_type == KVM_TYPE_Q4_0) go(d, std::integral_constant<int, KVM_TYPE_Q4_0>{});
                else go(d, std::integral_constant<int, KVM_TYPE_F16>{});
            };
            if (D == 256) go_d(std::integral_constant<int, 256>{});
            else go_d(std::integral_constant<int, 128>{});
            g.u.units = 0;
        }
    });
    KVM_LAUNCH_CHECK(st, what);
    return KVM_OK;
}
