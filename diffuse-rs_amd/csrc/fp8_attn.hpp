// fp8_attn.hpp -- what the attention kernels of DR_PRECISION_FP8 layers share
// (attn_fp8.hip, attn_fp8_wide.hip): loading and splitting query rows, the
// widening of codes, one key tile's scores, softmax and values, the output rows.
//
// With codes k, v and scales 2^ek, 2^ev of a position, and c = scale * log2 e:
//   s_j = c 2^ek_j (q . k_j)      p_j = exp2(s_j - m)      over visible j
//   out = sum_j p_j 2^ev_j v_j / sum_j p_j
// in one pass over the keys with a running maximum m and sum l in f32.
//
// Arithmetic.  Codes are exact in f16, so both products run on f16 MFMA with
// f32 accumulation (v_mfma_f32_32x32x16_f16 / 16x16x32):
// - Each query row is scaled by a power of two (largest magnitude to 2^14..2^15)
//   and split into PL planes of f16.  PL 2 (f32 rows): hi = f16(q), lo =
//   f16(q - hi), 22 bits.  PL 1 (bf16 rows in and out): the 8 bits of a bf16
//   are exact in f16.  The probabilities split likewise; with PL 1 they keep
//   f16's 11 bits, an eighth of the output's own rounding.
// - K's scale enters as its codes are widened: v_cvt_scalef32_pk_f16_fp8 takes
//   a power of two per lane, and a lane of the A operand is one key.  It is
//   taken relative to a K scale (kref), 2^7 up, which keeps every code exact to
//   scales 2^TK below it; 2^kref goes into the factor of the scores.
// - V's scale multiplies the planes of p, relative to the largest V scale met
//   so far (vref; the accumulators are rescaled when it rises): powers of two in
//   f16, down to 2^-TV; 2^vref is applied once at the end.  The planes end at
//   2^-24, so a weight so scaled is off by 2^-24 (one plane: 2^-25) at most, where
//   the row's largest is 2^P0 or more: by 2^-22 (2^-19) of that largest beside a
//   V row 2^TV larger, seen or not, and by 2^-34 (2^-35) among rows of one scale.
// - Scales further apart than that, which a cache need not have but may (a row of
//   1e30 must not cost queries that do not see it their bits), take a slower way
//   (FAR), on which a wave that has met them starts again; the common loop only
//   notes them (as branches of one loop that way cost every call 6-17 %).
//   A tile is walked again for each band of K scales, with the keys of the others
//   hidden.  V's scales go into the exponents of the weights, relative to a vref
//   of each row's own, so that a row's largest product is the measure of its
//   others (`apart`, from the first V tile that needs it).
// - m moves only when a score exceeds it by more than 2^MOVE, so p <= 2^(P0 +
//   MOVE) = 2^15 with p = exp2(s - m + P0), inside f16's range, and the
//   O rescale is skipped on almost every tile; out does not depend on m.  A
//   larger P0 keeps more of light weights, a smaller MOVE rescales more often:
//   P0 8 / 10 / 11 / 12, 256 bf16 rows x 16/8 heads of 256 in a window of 1024
//   17.4 / 18.1 / 18.2 / 18.5 us, 256 f32 rows x 16/2 heads of 512 over 4352 keys
//   94 / 95 / 92 / 99, 256 f32 rows x 32 heads of 128 over 768 13.5 / 13.6 / 13.6 / 13.8.
//
// S^T = K Q^T and O^T = V^T P^T: a lane owns one query column of both, so the
// softmax statistics are per lane, and with the keys of a tile assigned to A
// rows in the order of sigma() / kappa() a lane's scores are the very keys that
// its P operand needs; P never leaves registers.
//
// A key that a row may not see never reaches its output: its p is set to 0 and
// its codes are finite always (a row that held a NaN has codes 0 and the NaN in
// its scale byte, which is applied to visible keys only).  A row that sees no
// key ends 0 * (1 / 0) = NaN, like the reference (attention.rs:181-185).
#pragma once

#include "attn_common.hpp"
#include "fp8_common.hpp"

#include <type_traits>

#include <float.h>
#include <math.h>

namespace dr {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float P0 = 10.0f, MOVE = 5.0f;
constexpr int TK = 22;
template <int PL>
constexpr int TV = PL == 2 ? 12 : 16;
// Rows meet at 2^-LOW of themselves: sums of weights that start at 2^P0 would take
// values above 1e33 out of f32 before the division by the weights' sum.
constexpr int LOW = 18;
// How far vref may rise in all: the sums of a row that sees only the first tiles
// sink by as much (2^P0 or more at first; f32 holds them whole down to 2^-102).
constexpr int TV_RISE = 64;

// Whether a scale byte is one of values (not of a NaN's row or of zeros) and lies
// outside far .. 0 below ref.
__device__ __forceinline__ bool scale_far(int byte, int ref, int far) {
    return byte > 0 && byte != FP8_NAN && (byte > ref || byte < ref - far);
}
// The factor that widens K's codes of scale `byte` in the band that ends at ref.
__device__ __forceinline__ float band_scale(int byte, int ref) {
    return (unsigned)(byte - ref + TK) <= (unsigned)TK ? __uint_as_float((uint32_t)(byte - ref + 127 + 7) << 23) : 0.0f;
}
// LDS written by lanes of this wave, before others of it read it.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// The largest of 64 lanes' values, uniform: along each row of 16 lanes, then row to
// row, by DPP (a chain of 6 vector instructions; shuffles through LDS take 6 round
// trips).
__device__ __forceinline__ int wave_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));  // row_shr:1
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));  // row_shr:2
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));  // row_shr:4
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));  // row_shr:8
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));  // row_bcast:15
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));  // row_bcast:31
    return __builtin_amdgcn_readlane(x, 63);
}
// A band of K scales: bytes of values from ref - TK to ref, with NaN rows in the
// first band of a tile and rows of zeros in its last.
struct Band {
    int ref;
    bool first, last;
    __device__ __forceinline__ bool holds(int byte) const {
        return byte == FP8_NAN ? first : byte == 0 ? last : byte <= ref && byte >= ref - TK;
    }
};
// The power of two that brings a row's accumulators, the largest of them `big`, to
// about 2^16 where they are far from it (0: they are 0, or no number).
__device__ __forceinline__ int centre(float big) {
    const int e = (int)(__float_as_uint(big) >> 23) - 127;
    return big == 0.0f || e > 127 || (e >= 8 && e <= 24) ? 0 : 16 - e;
}

__device__ __forceinline__ f32x16 mfma(const f16x8& a, const f16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 codes -> f16, times 2^(exponent of scale)
__device__ __forceinline__ f16x8 widen(uint32_t w0, uint32_t w1, float scale) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w0, scale, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w0, scale, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w1, scale, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w1, scale, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// p - hi, hi widened on the way (one v_fma_mix_f32 each; the compiler makes two
// instructions of it)
__device__ __forceinline__ f32x2 residual(const f32x2& p, const f16x2& hi) {
    f32x2 r = {};
#if defined(__HIP_DEVICE_COMPILE__)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(hi), "v"(p[0]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(hi), "v"(p[1]));
#endif
    return r;
}

__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float((uint32_t)max(e, 0) << 23); }

// What every workgroup takes from the arguments, batch slot 0 included, is
// requested at its start in a few wide scalar loads with one wait; left to first
// uses, eight loads wait for each other (1 us of a call's 10).  The empty asm also
// keeps the compiler from choosing the slot by its address, which is one more.
__device__ __forceinline__ AttnSlot request_args(const AttnArgs& a) {
    AttnSlot S = a.slot[0];
    asm volatile("" : "+s"(S.q), "+s"(S.out), "+s"(S.qpos), "+s"(S.k), "+s"(S.vt), "+s"(S.klo), "+s"(S.nq), "+s"(S.nk),
                 "+s"(S.qpos0)
                 : "s"(a.n_batch), "s"(a.n_head_kv), "s"(a.group), "s"(a.hd), "s"(a.cap), "s"(a.q_rstride),
                   "s"(a.rowgroups), "s"(a.n_split), "s"(a.mg_split), "s"(a.mg_rowgroups), "s"(a.mg_hkv), "s"(a.c),
                   "s"(a.n_wg), "s"(a.window), "s"(a.prefix), "s"(a.o_rstride), "s"(a.qn_w), "s"(a.qb), "s"(a.rope),
                   "s"(a.q_bf16), "s"(a.o_bf16), "s"(a.mg_group));
    return S;
}

__device__ __forceinline__ int row_pos(const AttnSlot& S, int qi) { return S.qpos0 >= 0 ? S.qpos0 + qi : S.qpos[qi]; }

// Values d..d + 3 of a query row (0 past head_dim), f32.
template <int HD>
__device__ __forceinline__ f32x4 query4(const AttnArgs& a, const AttnSlot& S, size_t row, int d) {
    f32x4 y;
    if (a.q_bf16) {
        const uint16_t* q = static_cast<const uint16_t*>(S.q) + row + d;
        if (a.hd == HD) {  // (rows and heads start 8-byte aligned)
            const u32x2 w = gload<u32x2>(q);
            y = f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                      __uint_as_float(w[1] & 0xffff0000u)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = d + e < a.hd ? __uint_as_float((uint32_t)gload<uint16_t>(q + e) << 16) : 0.0f;
        }
    } else {
        const float* q = static_cast<const float*>(S.q) + row + d;
        if (a.hd == HD) {
            y = gload<f32x4>(q);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = d + e < a.hd ? gload<float>(q + e) : 0.0f;
        }
    }
    return y;
}

// Four values of a vector of head_dim parameters (0 past it).
__device__ __forceinline__ f32x4 param4(const float* w, int d, int hd) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = d + e < hd ? w[d + e] : 0.0f;
    return y;
}

// Values d0 .. d0 + 15 of a query row that LPR consecutive lanes hold, with the
// Q epilogue applied (forward.rs:291-310: bias, RMSNorm with f32 squares summed
// in f64, RoPE, whose partners d +- rot/2, rot/2 a multiple of 4, are loaded
// again).
template <int HD>
__device__ __forceinline__ void load_query(const AttnArgs& a, const AttnSlot& S, int qi, int head, int d0,
                                           f32x4 (&y)[4]) {
#pragma clang fp contract(off)
    constexpr int LPR = HD / 16;
    const size_t row = (size_t)qi * a.q_rstride + (size_t)head * a.hd;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = query4<HD>(a, S, row, d0 + 4 * i);
    if (!a.qb && !a.qn_w && !a.rope) return;
    const float* bias = a.qb ? a.qb + (size_t)head * a.hd : nullptr;
    if (bias)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += param4(bias, d0 + 4 * i, a.hd);
    float sc = 1.0f;
    if (a.qn_w) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float sq = y[i / 4][i % 4] * y[i / 4][i % 4];
            ss += (double)sq;
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        sc = 1.0f / (float)sqrt(ss / (double)a.hd + (double)a.qn_eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] * sc * param4(a.qn_w, d0 + 4 * i, a.hd);
    }
    if (a.rope) {
        const int half = a.rot / 2, pos = row_pos(S, qi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = d0 + 4 * i;
            if (d >= a.rot) continue;  // (rot is a multiple of 8)
            const int pd = d < half ? d + half : d - half, k = d < half ? d : pd;
            f32x4 x = query4<HD>(a, S, row, pd);
            if (bias) x += param4(bias, pd, a.hd);
            if (a.qn_w) x = x * sc * param4(a.qn_w, pd, a.hd);
            const float* t = a.rope + ((size_t)pos * half + k) * 2;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[i][e] = d < half ? rope_lo(y[i][e], x[e], t[2 * e], t[2 * e + 1])
                                   : rope_hi(x[e], y[i][e], t[2 * e], t[2 * e + 1]);
        }
    }
}

// The power of two that brings a row's largest magnitude to 2^14..2^15 (up, with
// the sign of c; 2^127 at most), and its inverse's exponent (the inverse itself may
// be subnormal); a row with a NaN or an infinity becomes NaN, and so does every row
// under a scale that is NaN.
template <int LPR>
__device__ __forceinline__ void query_scale(const AttnArgs& a, const f32x4 (&y)[4], float& up, int& down) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(y[e / 4][e % 4]) & 0x7fffffffu);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    const bool bad = top >= 0x7f800000u || a.c != a.c;
    const int ex = min(268 - (int)(top >> 23), 254);
    up = bad ? __uint_as_float(0x7fc00000u) : pow2_biased(ex);
    if (a.c < 0.0f) up = -up;
    down = bad ? 0 : 127 - ex;
}

// Values 8 h .. 8 h + 7 of a run, scaled, as f16 planes.
__device__ __forceinline__ void split8(const f32x4 (&y)[4], int h, float up, f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float z = y[2 * h + e / 4][e % 4] * up;
        hi[e] = (_Float16)z;
        lo[e] = (_Float16)(z - (float)hi[e]);
    }
}

// out[row] of packed row r, four values from d on
template <int HD>
__device__ __forceinline__ void write_out(const AttnArgs& a, const AttnSlot& S, int g, int r, int d, const f32x4& y) {
    const int qi = udiv(r, a.group, a.mg_group), head = g * a.group + (r - qi * a.group);
    const size_t o = (size_t)qi * a.o_rstride + (size_t)head * a.hd + d;
    if (a.o_bf16) {
        uint16_t* to = reinterpret_cast<uint16_t*>(S.out) + o;
        const bf16x4 b = {(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
        if (a.hd == HD) {
            *reinterpret_cast<bf16x4*>(to) = b;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < a.hd) to[e] = __builtin_bit_cast(uint16_t, (__bf16)y[e]);
        }
    } else if (a.hd == HD) {
        *reinterpret_cast<f32x4*>(S.out + o) = y;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.hd) S.out[o + e] = y[e];
    }
}

// The query rows r0 .. r0 + QR - 1 on their way to LDS: a thread takes 16 values
// of a row, all rows of a pass in flight at once.
template <int HD, int QR, int PL, int NT, int QP>
struct Fp8Queries {
    static constexpr int LPR = HD / 16, PER = NT / LPR, PASSES = (QR + PER - 1) / PER;  // lanes per row, rows per pass
    f32x4 y[PASSES][4];

    __device__ __forceinline__ void load(const AttnArgs& a, const AttnSlot& S, int g, int r0, int rows) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            // (a row past the last is the last again; lanes of a row agree)
            const int i = p * PER + (int)threadIdx.x / LPR, r = min(r0 + min(i, QR - 1), rows - 1);
            const int qi = udiv(r, a.group, a.mg_group);
            load_query<HD>(a, S, qi, g * a.group + r - qi * a.group, (int)threadIdx.x % LPR * 16, y[p]);
        }
    }
    // scaled by a power of two each (its inverse's exponent to srow), split into PL
    // planes of f16 in sq [PL][QR][QP]
    __device__ __forceinline__ void stage(const AttnArgs& a, _Float16* sq, int* srow) const {
        const int tid = threadIdx.x, d0 = tid % LPR * 16;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int i = p * PER + tid / LPR;
            float up;
            int down;
            query_scale<LPR>(a, y[p], up, down);
            if (i < QR) {
                if (tid % LPR == 0) srow[i] = down;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f16x8 hi, lo;
                    split8(y[p], h, up, hi, lo);
                    *reinterpret_cast<f16x8*>(sq + i * QP + d0 + 8 * h) = hi;
                    if constexpr (PL == 2) *reinterpret_cast<f16x8*>(sq + (QR + i) * QP + d0 + 8 * h) = lo;
                }
            }
        }
    }
};

// One row block's running state and the work of one key tile on it.  QR query
// rows (columns of the transposed products): 32, or 16.
template <int HD, int QR, int PL>
struct Fp8State {
    static constexpr int KB = QR == 32 ? 1 : 2;       // A blocks (32 or 16 keys) of a tile
    static constexpr int SK = QR == 32 ? 16 : 32;     // contraction of one MFMA
    static constexpr int NS = HD / SK;                // QK^T steps
    static constexpr int DB = HD / QR;                // row blocks of O^T
    static constexpr int SPL = 32 * QR / 64 / KB;     // scores per lane and A block: 16 or 4
    static constexpr int NP = SPL * KB;               // scores per lane: 16 or 8
    using Acc = std::conditional_t<QR == 32, f32x16, f32x4>;

    Acc o[DB];
    float m, l, kc;
    int kref, vref, vfirst;  // (vref: a row's own once `apart`; vfirst: where it rose from 0 to)
    bool apart, bad;  // (bad: scales too far apart without FAR, the state is worth nothing)
    float c;  // |c|, and the exponent of the inverse of the row's power of two
    int eq;

    __device__ __forceinline__ void init(float c_, int eq_) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < SPL; ++i) o[db][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
        kc = FLT_MIN;  // (before any stored key; never 0, a hidden score of -infinity has to stay one)
        kref = vref = vfirst = 0;
        apart = bad = false;
        c = fabsf(c_);
        eq = eq_;
    }

    // o times 2^e, |e| <= 252, in two steps
    __device__ __forceinline__ void scale(int e) {
        const float a = pow2_biased(e / 2 + 127), b = pow2_biased(e - e / 2 + 127);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= b;
    }

    // kb0, kb1: K's scale bytes of this lane's A rows (32 rows: the same twice);
    // vb: V's of key lane % 32; vs: 32 f16 of this wave in LDS.  kcodes(block,
    // step) and vcodes(row block, step): 8 codes as two dwords; query(plane,
    // step).  slow: some key may be hidden from some row, then see(i) tells of
    // the lane's i-th key (NP * half + i) whether its row sees it; kbyte(i), its
    // K scale byte, is asked where the tile has a NaN.  scored(next) is called once
    // K's codes are read.
    // With FAR: cap, where the K scales of this walk end (FP8_NAN: all); returns where
    // those of the tile's next walk end, 0 after its last.
    template <bool FAR, class KC, class VC, class Q, class See, class KByte, class Scored>
    __device__ __forceinline__ int tile(int cap, int kb0, int kb1, int vb, _Float16* vs, bool slow, KC kcodes, VC vcodes,
                                         Q query, See see, KByte kbyte, Scored scored) {
        bool nan = false;
        slow = __builtin_amdgcn_readfirstlane(slow);  // (uniform, and known to be: the masks stay behind a branch)
        const int lane = threadIdx.x & 63, half = lane / QR;
        // ---- scales: within TK of kref and TV of vref, as almost always?  (A NaN's
        // byte is above, that of a row of zeros below all others.)
        int next = 0;
        Band band{};
        bool banded = FAR && cap != FP8_NAN;
        if (__any((unsigned)(kb0 - kref + TK) > (unsigned)TK || (KB > 1 && (unsigned)(kb1 - kref + TK) > (unsigned)TK) ||
                  (unsigned)(vb - vref + TV<PL>) > (unsigned)TV<PL> || (FAR && (apart || banded)))) {
            const int k0 = kb0 > min(cap, FP8_NAN - 1) ? 0 : kb0, k1 = kb1 > min(cap, FP8_NAN - 1) ? 0 : kb1;
            const int kt = wave_max(max(k0, k1)), vt = wave_max(vb == FP8_NAN ? 0 : vb);
            nan = __any(kb0 == FP8_NAN || kb1 == FP8_NAN || vb == FP8_NAN);
            if (kt > kref || __any(scale_far(k0, kref, TK) || scale_far(k1, kref, TK)) || (FAR && kt > 0)) {
                kref = kt;
                kc = __builtin_fmaxf(ldexpf(c, eq + kref - 127 - 7), FLT_MIN);
            }
            const bool steep = vfirst > 0 && vt > vfirst + TV_RISE;
            if constexpr (FAR) {
                next = wave_max(max(scale_far(k0, kref, TK) ? k0 : 0, scale_far(k1, kref, TK) ? k1 : 0));
                banded = banded || next > 0;
                band = {kref, cap == FP8_NAN, next == 0};
            } else if (__builtin_expect(__any(scale_far(k0, kref, TK) || scale_far(k1, kref, TK) ||
                                              scale_far(vb, max(vref, vt), TV<PL>)) || steep, 0)) {
                bad = true;
            }
            if (!(FAR && apart) && vt > vref && !steep) {
                if (vref > 0) {
                    const float f = pow2_biased(vref - vt + 127);
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] *= f;
                } else {  // (o is 0)
                    vfirst = vt;
                }
                vref = vt;
            }
            if constexpr (FAR) apart = apart || __any(scale_far(vb, vref, TV<PL>));
            if (FAR && apart) {
                float big = 0.0f;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < SPL; ++i) big = __builtin_fmaxf(big, fabsf(o[db][i]));
#pragma unroll
                for (int off = QR; off < 64; off <<= 1) big = __builtin_fmaxf(big, __shfl_xor(big, off));
                const int up = centre(big);
                scale(up);
                vref = big == 0.0f ? 0 : vref - up;
            }
        }
        const bool far = FAR && __builtin_amdgcn_readfirstlane(apart);
        if (lane < 32)
            vs[lane] = (_Float16)(far ? (float)vb : vb == FP8_NAN ? INFINITY : pow2_biased(vb - vref + 127));

        // ---- scores of this lane's column
        float s[NP];
        Acc acc[KB] = {};
        const float ks0 = band_scale(kb0, kref), ks1 = KB > 1 ? band_scale(kb1, kref) : ks0;
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const u32x2 w = kcodes(kb, st);
                const f16x8 k8 = widen(w[0], w[1], kb ? ks1 : ks0);
#pragma unroll
                for (int p = 0; p < PL; ++p) acc[kb] = mfma(k8, query(p, st), acc[kb]);
            }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < SPL; ++i) s[kb * SPL + i] = acc[kb][i];
        if constexpr (FAR) next = __builtin_amdgcn_readfirstlane(next);
        scored(next);

        // ---- masks: scores the row may not use
        uint32_t hidden = 0;
        if (FAR && __builtin_amdgcn_readfirstlane(banded)) {
            slow = true;
#pragma unroll
            for (int i = 0; i < NP; ++i) hidden |= band.holds(kbyte(i)) ? 0 : 1u << i;
        }
        if (slow) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool ok = see(i) && !(hidden >> i & 1);
                hidden |= ok ? 0 : 1u << i;
                s[i] = ok ? s[i] : -INFINITY;
            }
        }
        if (nan)
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (!(hidden >> i & 1) && kbyte(i) == FP8_NAN) s[i] = NAN;

        // ---- running maximum (moved rarely), probabilities, sum
        float top = s[0];
#pragma unroll
        for (int i = 1; i < NP; ++i) top = __builtin_fmaxf(top, s[i]);
        const float ts = top == -INFINITY ? -INFINITY : top * kc;
        float kcl = kc, l_far = 0.0f;
        if (__any(ts > m + MOVE) || far) {
            float nm = ts;
#pragma unroll
            for (int off = QR; off < 64; off <<= 1) nm = __builtin_fmaxf(nm, __shfl_xor(nm, off));
            nm = nm > m + MOVE ? nm : m;
            float f = m == nm ? 1.0f : __builtin_amdgcn_exp2f(m - nm);
            l *= f;
            if (far) {
                // the weights' sum, and V's scales into their exponents, 2^15 at most
                const float off = P0 - (nm == -INFINITY ? 0.0f : nm);
                float most = -INFINITY;
                wave_lds();
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float byte = (float)vs[NP * half + i];
                    s[i] = __builtin_fmaf(s[i], kc, off);
                    l_far += __builtin_amdgcn_exp2f(s[i]);
                    if (byte != (float)FP8_NAN) most = __builtin_fmaxf(most, s[i] + (byte - (float)vref));
                }
                l_far += l;
#pragma unroll
                for (int o2 = QR; o2 < 64; o2 <<= 1) most = __builtin_fmaxf(most, __shfl_xor(most, o2));
                const int rise = most > P0 + MOVE ? (int)__builtin_fminf(ceilf(most - P0), 252.0f) : 0;
                vref += rise;
                f *= pow2_biased(127 - rise / 2) * pow2_biased(127 - (rise - rise / 2));
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float byte = (float)vs[NP * half + i];
                    s[i] = byte == (float)FP8_NAN && s[i] != -INFINITY ? NAN : s[i] + (byte - (float)vref);
                }
                wave_lds();
                if (lane < 32) vs[lane] = (_Float16)1.0f;
                kcl = 1.0f;
            }
            if (__any(m != -INFINITY))  // (else o is 0)
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db] *= f;
            m = nm;
        }
        const float off = far || m == -INFINITY ? far ? 0.0f : P0 : P0 - m;
        wave_lds();
        f16x8 ph[NP / 8], pl[NP / 8];
        f16x8 sc[NP / 8];
#pragma unroll
        for (int i = 0; i < NP / 8; ++i) sc[i] = *reinterpret_cast<const f16x8*>(vs + NP * half + 8 * i);
        if (slow)  // (a hidden key's p is 0; a scale of infinity would still make it NaN)
#pragma unroll
            for (int i = 0; i < NP; ++i) sc[i / 8][i % 8] = hidden >> i & 1 ? (_Float16)0.0f : sc[i / 8][i % 8];
#pragma unroll
        for (int i = 0; i < NP; i += 2) {
            const f32x2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], kcl, off)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], kcl, off))};
            const f16x2 hi = __builtin_convertvector(p, f16x2);
            if constexpr (PL == 1) {
                // the sum is of the weights that the product takes
                l = __builtin_amdgcn_fdot2(hi, f16x2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
            } else {
                l += p[0];
                l += p[1];
                const f32x2 r = residual(p, hi);
                const f16x2 lo = __builtin_convertvector(r, f16x2);
                pl[i / 8][i % 8] = lo[0];
                pl[i / 8][i % 8 + 1] = lo[1];
            }
            ph[i / 8][i % 8] = hi[0];
            ph[i / 8][i % 8 + 1] = hi[1];
        }
#pragma unroll
        for (int i = 0; i < NP / 8; ++i) {
            ph[i] *= sc[i];
            if constexpr (PL == 2) pl[i] *= sc[i];
        }
        if (far) l = l_far;
        // ---- O^T += V^T P^T
        constexpr int DG = DB < 4 ? DB : 4;  // row blocks in turn: their MFMAs do not wait for each other
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += DG)
#pragma unroll
            for (int st = 0; st < NP / 8; ++st) {
                f16x8 v8[DG];
#pragma unroll
                for (int k = 0; k < DG; ++k) {
                    const u32x2 w = vcodes(d0 + k, st);
                    v8[k] = widen(w[0], w[1], 1.0f);
                    o[d0 + k] = mfma(v8[k], ph[st], o[d0 + k]);
                }
                if constexpr (PL == 2)
#pragma unroll
                    for (int k = 0; k < DG; ++k) o[d0 + k] = mfma(v8[k], pl[st], o[d0 + k]);
            }
        // (the next tile's V scales are written after this tile's reads)
        wave_lds();
        return FAR ? next : 0;
    }

    // l over the lanes that share a column
    __device__ __forceinline__ float row_sum() const {
        float t = l;
#pragma unroll
        for (int off = QR; off < 64; off <<= 1) t += __shfl_xor(t, off);
        return t;
    }
    // o's weight next to a state of maximum M, 2^vref (V's common factor) included,
    // and 2^-LOW, as for the sums: two factors, since for the smallest rows their
    // product is subnormal, which would cost o's bits (1e-36: all but 7)
    __device__ __forceinline__ f32x2 weight(float M) const {
        const int e = vref - 127 - LOW;
        const float w = m == -INFINITY ? (l != l ? l : 0.0f) : __builtin_amdgcn_exp2f(m - M);
        return f32x2{w * pow2_biased(e / 2 + 127), pow2_biased(e - e / 2 + 127)};
    }
    // the dim of o[db][i], i a multiple of 4: four consecutive dims from there
    __device__ static __forceinline__ int dim(int db, int i, int half) {
        return QR == 32 ? 32 * db + 2 * i + 4 * half : 16 * db + 4 * half;
    }
};

// The position of a row that the whole wave agrees on.
__device__ __forceinline__ int uniform_pos(const AttnSlot& S, int qi) {
    return __builtin_amdgcn_readfirstlane(row_pos(S, qi));
}

// Whether a tile holds only keys that every row at positions q_lo..q_hi sees.
__device__ __forceinline__ bool tile_visible(const AttnArgs& a, int nk, int t, int q_lo, int q_hi) {
    return 32 * t + 32 <= nk &&
           (a.window < 0 || (q_hi - 32 * t < a.window && 32 * t + 31 - q_lo < a.window)) &&
           (a.prefix < 0 || q_lo >= a.prefix || 32 * t + 31 <= q_lo);
}

// The key tiles that rows at positions q_lo..q_hi can see.
__device__ __forceinline__ void row_tiles(const AttnArgs& a, int nk, int q_lo, int q_hi, int& lo, int& hi) {
    lo = 0;
    hi = (nk + 31) / 32;
    if (a.window >= 0) band_tile_range(nk, a.window, q_lo, q_hi, lo, hi);
    if (a.prefix >= 0 && q_hi < a.prefix) hi = min(hi, q_hi / 32 + 1);
    hi = max(lo, hi);
}

// A workgroup of an 8 bit attention launch: its place in the grid.  Each XCD
// (the hardware deals workgroups round robin over the 8) takes a contiguous run
// of (batch slot, KV head, row group, key split), splits fastest: the splits of a
// row group share its query rows in an L2, and the joins are spread over the XCDs
// (with row groups fastest they ended on the XCD of the last split: 64 joins of 64
// rows of 512 dims, 4 splits, took 20 us instead of 13).
struct Fp8Place {
    int rg, split, g, b;
    bool ok;
    __device__ __forceinline__ explicit Fp8Place(const AttnArgs& a) {
        const int per = (a.n_wg + 7) / 8;
        int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
        ok = (int)(blockIdx.x >> 3) < per && id < a.n_wg;
        const int t = a.n_split > 1 ? udiv(id, a.n_split, a.mg_split) : id;
        split = id - t * a.n_split;
        const int u = udiv(t, a.rowgroups, a.mg_rowgroups);
        rg = a.rowgroups - 1 - (t - u * a.rowgroups);  // (under a causal prefix the last see the most keys)
        b = udiv(u, a.n_head_kv, a.mg_hkv);
        g = u - b * a.n_head_kv;
    }
};
inline unsigned fp8_grid(const AttnArgs& a) { return (unsigned)((a.n_wg + 7) / 8 * 8); }

// Key splits.  Each workgroup has stored the states of its rows r0 .. r0 + nr - 1
// with agent-scope accesses; it waits until they are complete, and one thread
// takes the row group's ticket.  The one that draws n_split - 1 is the last: the
// others' stores are complete and its agent-scope loads see them.  It joins the
// splits in an order of its own (the same bits whichever comes last), writes the
// rows and resets the ticket for the next call.  No workgroup waits for another.
// so: LDS of NT * 6 floats that nobody reads any more; stick: one int in LDS.
// (Byte offsets of the workspace fit 32 bits: the host checks.)
template <int HD, int NT>
__device__ __forceinline__ void fp8_join(const AttnArgs& a, const AttnSlot& S, const Fp8Place& at, int r0, int nr,
                                         float* so, int* stick) {
    const int tid = threadIdx.x, items = nr * (HD / 4);
    const size_t prow0 = ((size_t)at.b * a.n_head_kv + at.g) * a.part_rows + r0;
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.part_o, 0xffffffffu);
    const __amdgpu_buffer_rsrc_t rm = make_rsrc(a.part_ml, 0xffffffffu);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* const tk = a.ticket + (at.b * a.n_head_kv + at.g) * a.rowgroups + at.rg;
    if (tid == 0) *stick = __hip_atomic_fetch_add(tk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*stick != a.n_split - 1) return;
    if (tid == 0) __hip_atomic_store(tk, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Few rows leave threads over: `share` threads take an item's splits (thread
    // k of them takes splits k, k + share, ...), so that all loads of a wide
    // split are in flight together; their states join through LDS.
    // Many rows: a thread takes several items at once, 16 loads in flight.
    auto many = [&](auto ni, auto ns) __attribute__((always_inline)) {
        constexpr int NI = decltype(ni)::value, NS = decltype(ns)::value;
        for (int p = tid; p < items; p += NI * NT) {
            float Mx[NI], L[NI];
            f32x4 acc[NI][1];
#pragma unroll
            for (int q = 0; q < NI; ++q) {
                Mx[q] = -INFINITY;
                L[q] = 0.0f;
                acc[q][0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            for (int s0 = 0; s0 < a.n_split; s0 += NS) {
                float m[NI][NS], l[NI][NS];
                f32x4 o[NI][NS][1];
#pragma unroll
                for (int q = 0; q < NI; ++q) {
                    const int it = min(p + q * NT, items - 1);
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const size_t row = (size_t)min(s0 + j, a.n_split - 1) * plane + prow0 + it / (HD / 4);
                        const float2 ml = load2_sc1(rm, (int)(row * 8));
                        o[q][j][0] = load_sc1(ro, (int)((row * HD + it % (HD / 4) * 4) * 4));
                        m[q][j] = s0 + j < a.n_split ? ml.x : -INFINITY;
                        l[q][j] = ml.y;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // (every load above before any wait)
#pragma unroll
                for (int q = 0; q < NI; ++q) merge_split_states<NS, 1>(Mx[q], L[q], acc[q], m[q], l[q], o[q]);
            }
#pragma unroll
            for (int q = 0; q < NI; ++q) {
                const int it = p + q * NT;
                if (it < items)
                    write_out<HD>(a, S, at.g, r0 + it / (HD / 4), it % (HD / 4) * 4, acc[q][0] * (1.0f / L[q]));
            }
        }
    };
    if (items >= 2 * NT) {
        if (a.n_split <= 4)
            many(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
        else
            many(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
        return;
    }
    int share = 1;
    while (2 * share * items <= NT) share *= 2;
    for (int p = tid; p < share * items; p += NT) {
        const int k = p / items, it = p - k * items, i = it / (HD / 4), d = it % (HD / 4) * 4;
        float Mx = -INFINITY, L = 0.0f;
        f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int s0 = k; s0 < a.n_split; s0 += 8 * share) {
            float m[8], l[8];
            f32x4 o8[8][1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int sp = s0 + j * share;
                const size_t row = (size_t)min(sp, a.n_split - 1) * plane + prow0 + i;
                const float2 ml = load2_sc1(rm, (int)(row * 8));
                o8[j][0] = load_sc1(ro, (int)((row * HD + d) * 4));
                m[j] = sp < a.n_split ? ml.x : -INFINITY;
                l[j] = ml.y;
            }
            __builtin_amdgcn_sched_barrier(0);  // (every load above before any wait)
            merge_split_states<8, 1>(Mx, L, acc, m, l, o8);
        }
        if (share == 1) {
            write_out<HD>(a, S, at.g, r0 + i, d, acc[0] * (1.0f / L));
        } else {
            float* t = so + p * 6;
            t[0] = Mx;
            t[1] = L;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[2 + e] = acc[0][e];
        }
    }
    if (share == 1) return;
    __syncthreads();
    if (tid < items) {
        float Mx = -INFINITY, L = 0.0f;
        f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int k = 0; k < share; ++k) {
            const float* t = so + (k * items + tid) * 6;
            const float m[1] = {t[0]}, l[1] = {t[1]};
            const f32x4 w[1][1] = {{{t[2], t[3], t[4], t[5]}}};
            merge_split_states<1, 1>(Mx, L, acc, m, l, w);
        }
        write_out<HD>(a, S, at.g, r0 + tid / (HD / 4), tid % (HD / 4) * 4, acc[0] * (1.0f / L));
    }
}

// The end of a workgroup of NW waves on one block of QR rows: their states meet
// in LDS, the rows leave, or, with key splits, join the other splits'.  LDS: so [NW][QR][HD + 4] floats, sm and sl [NW][QR], sr
// [2][QR], stick one int; so may lie over what the waves read before (a barrier precedes).
template <int HD, int QR, int PL, int NW>
__device__ __forceinline__ void fp8_finish(const AttnArgs& a, const AttnSlot& S, const Fp8Place& at,
                                           const Fp8State<HD, QR, PL>& st, int r0, float* so, float* sm,
                                           float* sl, float* sr, int* stick) {
    using T = Fp8State<HD, QR, PL>;
    constexpr int OP = HD + 4, NT = NW * 64;
    const int tid = threadIdx.x, wave = tid >> 6, col = (tid & 63) % QR, half = (tid & 63) / QR;
    const float lt = st.row_sum();
    if (half == 0) {
        sm[wave * QR + col] = st.m;
        sl[wave * QR + col] = lt;
    }
    __syncthreads();
    float M = sm[col];
#pragma unroll
    for (int k = 1; k < NW; ++k) M = __builtin_fmaxf(M, sm[k * QR + col]);
    if (tid < QR) {  // the row's maximum and sum over the waves
        float L = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float mw = sm[k * QR + col], lw = sl[k * QR + col];
            L += mw == -INFINITY ? (lw != lw ? lw : 0.0f) : lw * __builtin_amdgcn_exp2f(mw - M - (float)LOW);
        }
        sr[col] = M;
        sr[QR + col] = L;
    }
    const f32x2 f = st.weight(M);
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
        for (int i = 0; i < T::SPL; i += 4)
            *reinterpret_cast<f32x4*>(so + (wave * QR + col) * OP + T::dim(db, i, half)) =
                f32x4{st.o[db][i], st.o[db][i + 1], st.o[db][i + 2], st.o[db][i + 3]} * f[0] * f[1];
    __syncthreads();
    const int nr = min(QR, S.nq * a.group - r0), items = nr * (HD / 4);
    // four values of row i, relative to its maximum
    auto joined = [&](int i, int d) __attribute__((always_inline)) {
        f32x4 acc = *reinterpret_cast<const f32x4*>(so + i * OP + d);
#pragma unroll
        for (int k = 1; k < NW; ++k) acc += *reinterpret_cast<const f32x4*>(so + (k * QR + i) * OP + d);
        return acc;
    };
    if (a.n_split == 1) {
        for (int p = tid; p < items; p += NT) {
            const int i = p / (HD / 4), d = p % (HD / 4) * 4;
            write_out<HD>(a, S, at.g, r0 + i, d, joined(i, d) * (1.0f / sr[QR + i]));
        }
        return;
    }

    // ---- key splits: this workgroup's states
    const size_t prow0 = ((size_t)at.b * a.n_head_kv + at.g) * a.part_rows + r0;
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.part_o, 0xffffffffu);
    const __amdgpu_buffer_rsrc_t rm = make_rsrc(a.part_ml, 0xffffffffu);
    for (int p = tid; p < items; p += NT) {
        const int i = p / (HD / 4), d = p % (HD / 4) * 4;
        const f32x4 acc = joined(i, d);
        const size_t row = (size_t)at.split * plane + prow0 + i;
        store_sc1(ro, (int)((row * HD + d) * 4), acc);
        // (a NaN without any finite score must not pass for a row without keys)
        const float Mi = sr[i], L = sr[QR + i];
        if (d == 0) store2_sc1(rm, (int)(row * 8), L != L && Mi == -INFINITY ? 0.0f : Mi, L);
    }
    fp8_join<HD, NT>(a, S, at, r0, nr, so, stick);
}

}  // namespace
}  // namespace dr
