// attn_fp8.hip -- attention over a DR_PRECISION_FP8 cache layer (the format:
// fp8_common.hpp).
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
//   taken relative to the largest K scale met so far (kref), 2^7 up, which
//   keeps every code exact to scales 2^22 below it; 2^kref goes into the
//   factor of the scores.
// - V's scale multiplies p in f32, relative to the largest V scale met so far
//   (vref; the accumulators are rescaled when it rises); 2^vref is applied
//   once at the end.
// - m moves only when a score exceeds it by more than 2^MOVE, so p <= 2^(P0 +
//   MOVE) = 2^15 with p = exp2(s - m + P0), inside f16's range, and the
//   O rescale is skipped on almost every tile; out does not depend on m.
//
// S^T = K Q^T and O^T = V^T P^T: a lane owns one query column of both, so the
// softmax statistics are per lane, and with the keys of a tile assigned to A
// rows in the order of sigma() / kappa() a lane's scores are the very keys that
// its P operand needs; P never leaves registers.
//
// A workgroup owns QR packed rows of one KV head (row r = query * group + head
// in group, so a block spans few positions) and a range of 32-key tiles; its NW
// waves take tiles t, t + NW, ..., each with its own state, and merge through
// LDS.  Tiles come straight from memory into registers, one ahead: the planes
// hold a tile in operand order, so every load is one contiguous run.  Few
// workgroups split the keys further: each leaves its state in a workspace, and
// the last one of a row block to finish (an atomic ticket) joins them.
//
// A key that a row may not see never reaches its output: its p is set to 0 and
// its codes are finite always (a row that held a NaN has codes 0 and the NaN in
// its scale byte, which is applied to visible keys only).  A row that sees no
// key ends 0 * (1 / 0) = NaN, like the reference (attention.rs:181-185).
#include "attn_common.hpp"
#include "fp8_common.hpp"

#include <algorithm>
#include <type_traits>

#include <float.h>

#include <math.h>

namespace dr {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float P0 = 8.0f, MOVE = 7.0f;
template <int HD, int QR, int PL, int NW>
struct Fp8Geo {
    static constexpr int KB = QR == 32 ? 1 : 2;       // A blocks (32 or 16 keys) of a tile
    static constexpr int SK = QR == 32 ? 16 : 32;     // contraction of one MFMA
    static constexpr int NS = HD / SK;                // QK^T steps
    static constexpr int DB = HD / QR;                // row blocks of O^T
    static constexpr int SPL = 32 * QR / 64 / KB;     // scores per lane and A block: 16 or 4
    static constexpr int NP = SPL * KB;               // scores per lane: 16 or 8
    static constexpr int KCH = HD * 32 / 16 / 64;     // 16-byte K pieces per lane and tile
    static constexpr int VW = HD * 32 / 4 / 64;       // dwords of V per lane and tile
    // Head dim 512: the query planes (128 registers) are read from LDS as they
    // are multiplied, for the registers' sake.
    static constexpr bool BIG = HD > 256;
    static constexpr int QP = HD + 8;                 // f16 pitch of a staged query row
    static constexpr int OP = HD + 4;                 // f32 pitch of a merged row
    static constexpr size_t Q_BYTES = (size_t)PL * QR * QP * 2;
    static constexpr size_t O_BYTES = (size_t)NW * QR * OP * 4;
    static constexpr size_t BODY = O_BYTES > Q_BYTES ? O_BYTES : Q_BYTES;
    // then: per-row scales, wave states, V scales (f16) of each wave's tile, the ticket
    static constexpr size_t LDS = BODY + QR * 4 + 2 * NW * QR * 4 + NW * 32 * 2 + 16;
};

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

__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float((uint32_t)max(e, 0) << 23); }

// dword w of p, as loaded bytes
__device__ __forceinline__ int byte_of(const u32x4& w, int i) { return (int)(w[i / 4] >> (8 * (i % 4))) & 255; }

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

// The Q epilogue (forward.rs:291-310) on values d0..d0 + 15 of a query row that
// HD / 16 consecutive lanes hold: bias, RMSNorm (f32 squares summed in f64),
// RoPE, whose partners d +- rot/2 (rot/2 a multiple of 4) are loaded again.
template <int HD>
__device__ __forceinline__ void query_epilogue(const AttnArgs& a, const AttnSlot& S, size_t row, int head, int pos,
                                               int d0, f32x4 (&y)[4]) {
#pragma clang fp contract(off)
    const float* bias = a.qb ? a.qb + (size_t)head * a.hd : nullptr;
    if (bias)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += param4(bias, d0 + 4 * i, a.hd);
    float sc = 1.0f;
    if (a.qn_w) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float sq = y[i][e] * y[i][e];
                ss += (double)sq;
            }
#pragma unroll
        for (int o = HD / 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        sc = 1.0f / (float)sqrt(ss / (double)a.hd + (double)a.qn_eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] * sc * param4(a.qn_w, d0 + 4 * i, a.hd);
    }
    if (a.rope) {
        const int half = a.rot / 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = d0 + 4 * i;
            if (d >= a.rot) continue;  // (rot is a multiple of 8)
            const int pd = d < half ? d + half : d - half, j = d < half ? d : pd;
            f32x4 x = query4<HD>(a, S, row, pd);
            if (bias) x += param4(bias, pd, a.hd);
            if (a.qn_w) x = x * sc * param4(a.qn_w, pd, a.hd);
            const float* t = a.rope + ((size_t)pos * half + j) * 2;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[i][e] = d < half ? rope_lo(y[i][e], x[e], t[2 * e], t[2 * e + 1])
                                   : rope_hi(x[e], y[i][e], t[2 * e], t[2 * e + 1]);
        }
    }
}

// The query rows r0 .. r0 + ROWS - 1: with the epilogue applied, scaled by a
// power of two each (inverse to srow), split into PL planes of f16 in sq
// [PL][ROWS][QP].  A thread takes 16 values of a row, all rows of a pass in
// flight at once.
template <int HD, int ROWS, int PL, int NT, int QP>
__device__ __forceinline__ void stage_queries(const AttnArgs& a, const AttnSlot& S, int g, int r0, int rows,
                                              _Float16* sq, float* srow) {
    constexpr int LPR = HD / 16, PER = NT / LPR;  // lanes per row, rows per pass
    const int tid = threadIdx.x, d0 = tid % LPR * 16;
#pragma unroll
    for (int p = 0; p < (ROWS + PER - 1) / PER; ++p) {
        const int i = p * PER + tid / LPR;
        // (a row past the last is the last again; lanes of a row agree)
        const int r = min(r0 + min(i, ROWS - 1), rows - 1), qi = r / a.group, head = g * a.group + r - qi * a.group;
        const size_t row = (size_t)qi * a.q_rstride + (size_t)head * a.hd;
        f32x4 y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = query4<HD>(a, S, row, d0 + 4 * e);
        if (a.qb || a.qn_w || a.rope) query_epilogue<HD>(a, S, row, head, a.rope ? row_pos(S, qi) : 0, d0, y);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(y[e / 4][e % 4]) & 0x7fffffffu);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        // 2^14 <= |largest| * up < 2^15; a row with a NaN or an infinity gives NaN
        const bool bad = top >= 0x7f800000u;
        const int ex = min(268 - (int)(top >> 23), 254);
        float up = bad ? __uint_as_float(0x7fc00000u) : pow2_biased(ex);
        if (a.c < 0.0f) up = -up;
        if (i < ROWS) {
            if (tid % LPR == 0) srow[i] = pow2_biased(bad ? 127 : 254 - ex);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f16x8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = y[2 * h + e / 4][e % 4] * up;
                    hi[e] = (_Float16)z;
                    lo[e] = (_Float16)(z - (float)hi[e]);
                }
                *reinterpret_cast<f16x8*>(sq + i * QP + d0 + 8 * h) = hi;
                if constexpr (PL == 2) *reinterpret_cast<f16x8*>(sq + (ROWS + i) * QP + d0 + 8 * h) = lo;
            }
        }
    }
}


// out[row] of packed row r, four values from d on
template <int HD>
__device__ __forceinline__ void write_out(const AttnArgs& a, const AttnSlot& S, int g, int r, int d, const f32x4& y) {
    const int qi = r / a.group, head = g * a.group + (r - qi * a.group);
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

template <int HD, int QR, int PL, int NW>
__global__ __launch_bounds__(NW * 64) void attn_fp8_kernel(const AttnArgs a) {
    using G = Fp8Geo<HD, QR, PL, NW>;
    using Acc = std::conditional_t<QR == 32, f32x16, f32x4>;
    extern __shared__ __align__(16) char lds[];
    _Float16* const sq = reinterpret_cast<_Float16*>(lds);                 // [PL][QR][QP]
    float* const so = reinterpret_cast<float*>(lds);                       // [NW][QR][OP], after the key loop
    float* const srow = reinterpret_cast<float*>(lds + G::BODY);           // [QR]
    float* const sm = srow + QR;                                           // [NW][QR]
    float* const sl = sm + NW * QR;                                        // [NW][QR]
    _Float16* const svs = reinterpret_cast<_Float16*>(sl + NW * QR);       // [NW][32]
    int* const stick = reinterpret_cast<int*>(svs + NW * 32);

    // Workgroup -> (batch slot, KV head, key split, row block): each XCD (the
    // hardware deals workgroups round robin over the 8) takes a contiguous run,
    // so the row blocks that read the same keys share an L2.
    const int per = (a.n_wg + 7) / 8;
    int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= a.n_wg) return;
    const int rb = id % a.rowgroups;
    id /= a.rowgroups;
    const int split = id % a.n_split;
    id /= a.n_split;
    const int g = id % a.n_head_kv, b = id / a.n_head_kv;
    const AttnSlot& S = a.slot[b];
    const int rows = S.nq * a.group, r0 = rb * QR;
    if (r0 >= rows) return;  // (a shorter pass of the batch)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane % QR, half = lane / QR;  // query column; 0..1 (0..3 with 16 rows)

    // ---- the key tiles this workgroup's rows can see
    const int q_lo = row_pos(S, r0 / a.group), q_hi = row_pos(S, (min(r0 + QR, rows) - 1) / a.group);
    const int my_r = min(r0 + col, rows - 1);
    const int my_pos = row_pos(S, my_r / a.group);
    int kt_lo = 0, kt_hi = (S.nk + 31) / 32;
    if (a.window >= 0) band_tile_range(S.nk, a.window, q_lo, q_hi, kt_lo, kt_hi);
    if (a.prefix >= 0 && q_hi < a.prefix) kt_hi = min(kt_hi, q_hi / 32 + 1);
    int t0, t1;
    split_tile_range(kt_lo, max(kt_lo, kt_hi), a.n_split, split, t0, t1);

    const uint8_t* const kbase = reinterpret_cast<const uint8_t*>(S.k) + fp8_tile(g, a.cap, 0, HD);
    const uint8_t* const vbase = reinterpret_cast<const uint8_t*>(S.vt) + fp8_tile(g, a.cap, 0, HD);
    const uint8_t* const sbase = reinterpret_cast<const uint8_t*>(S.klo) + fp8_scale_tile(g, a.cap, 0);
    const int last_tile = a.cap / 32 - 1;

    struct Tile {
        u32x4 k[G::KCH];
        uint32_t v[G::VW];
        int kb, vb;  // scale bytes: K's of this lane's A row (16 rows: of both blocks, 8 bits each), V's of key lane % 32
    };
    // K and scales, then V: a step refills K's registers once its scores are
    // formed and V's once its product is, so the loads run under the rest of the
    // step and a tile ahead costs no registers.  (A tile past the plane's end,
    // which nobody multiplies, is its last one.)
    auto fetch_k = [&](int t, Tile& x) __attribute__((always_inline)) {
        t = min(t, last_tile);
        const uint8_t* kt = kbase + (size_t)t * 32 * HD;
        const uint8_t* st = sbase + (size_t)t * 64;
        if constexpr (QR == 32) {
            const int key = sigma(col);
            x.kb = gload<uint8_t>(st + key);
            x.vb = gload<uint8_t>(st + 32 + (lane & 31));
#pragma unroll
            for (int j = 0; j < G::KCH; ++j) x.k[j] = gload<u32x4>(kt + (2 * j + half) * 512 + key * 16);
        } else {
            x.kb = (int)gload<uint8_t>(st + kappa(col)) | (int)gload<uint8_t>(st + kappa(16 + col)) << 8;
            x.vb = gload<uint8_t>(st + 32 + (lane & 31));
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key = kappa(16 * kb + col);
#pragma unroll
                for (int j = 0; j < G::KCH / 2; ++j)
                    x.k[kb * (G::KCH / 2) + j] = gload<u32x4>(kt + (4 * j + half) * 512 + key * 16);
            }
        }
    };
    auto fetch_v = [&](int t, Tile& x) __attribute__((always_inline)) {
        const uint8_t* vt = vbase + (size_t)min(t, last_tile) * 32 * HD;
        if constexpr (QR == 32) {
#pragma unroll
            for (int db = 0; db < G::DB; ++db) {
                const u32x4 w = gload<u32x4>(vt + (32 * db + col) * 32 + half * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.v[4 * db + e] = w[e];
            }
        } else {
#pragma unroll
            for (int db = 0; db < G::DB; ++db) {
                const u32x2 w = gload<u32x2>(vt + (16 * db + col) * 32 + half * 8);
                x.v[2 * db] = w[0];
                x.v[2 * db + 1] = w[1];
            }
        }
    };

    Tile x;
    const int t_first = t0 + wave;
    if (t_first < t1) {  // (in flight while the query rows are staged)
        fetch_k(t_first, x);
        fetch_v(t_first, x);
    }

    // ---- the query rows
    stage_queries<HD, QR, PL, NW * 64, G::QP>(a, S, g, r0, rows, sq, srow);
    __syncthreads();
    auto query = [&](int p, int s) __attribute__((always_inline)) {
        // K piece j of a lane holds 16 values, steps 2j and 2j + 1
        const int d = ((64 / QR) * (s / 2) + half) * 16 + s % 2 * 8;
        return *reinterpret_cast<const f16x8*>(sq + (p * QR + col) * G::QP + d);
    };
    f16x8 q[PL][G::BIG ? 1 : G::NS];
    if constexpr (!G::BIG)
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int s = 0; s < G::NS; ++s) q[p][s] = query(p, s);
    const float cq = fabsf(a.c) * srow[col];

    Acc o[G::DB];
#pragma unroll
    for (int db = 0; db < G::DB; ++db)
#pragma unroll
        for (int i = 0; i < G::SPL; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, l = 0.0f, kc = 0.0f;
    int kref = 0, vref = 0;
    _Float16* const my_vs = svs + wave * 32;

    auto step = [&](int t, Tile& x) __attribute__((always_inline)) {
        // ---- scales: relative to the largest so far
        bool slow = !(32 * t + 32 <= S.nk && (a.window < 0 || (q_hi - 32 * t < a.window && 32 * t + 31 - q_lo < a.window)) &&
                      (a.prefix < 0 || q_lo >= a.prefix || 32 * t + 31 <= q_lo));
        const int kb0 = QR == 32 ? x.kb : x.kb & 255, kb1 = QR == 32 ? x.kb : x.kb >> 8;
        if (__any(max(kb0, kb1) > kref || x.vb > vref)) {
            // (a NaN's byte is larger than any other, so a tile with one comes here)
            const int k0 = kb0 == FP8_NAN ? 0 : kb0, k1 = kb1 == FP8_NAN ? 0 : kb1;
            int kt = max(k0, k1), vt = x.vb == FP8_NAN ? 0 : x.vb;
            slow = slow || __any(kb0 == FP8_NAN || kb1 == FP8_NAN || x.vb == FP8_NAN);
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                kt = max(kt, __shfl_xor(kt, off));
                vt = max(vt, __shfl_xor(vt, off));
            }
            kref = max(kref, kt);
            // (never 0: a hidden score of -infinity has to stay one)
            kc = ldexpf(cq, kref - 127 - 7);
            kc = kc < FLT_MIN ? FLT_MIN : kc;
            if (vt > vref) {
                const float f = pow2_biased(vref - vt + 127);
#pragma unroll
                for (int db = 0; db < G::DB; ++db) o[db] *= f;
                vref = vt;
            }
        }
        // V's scales, f16 (the smallest powers of two are f16's subnormals)
        if (lane < 32) my_vs[lane] = (_Float16)(x.vb == FP8_NAN ? INFINITY : pow2_biased(x.vb - vref + 127));
        const float ks0 = pow2_biased(min(kb0 - kref, 0) + 127 + 7), ks1 = pow2_biased(min(kb1 - kref, 0) + 127 + 7);

        // ---- scores of this lane's column: key 16 half + i (32 rows) or 8 half + i
        float s[G::NP];
        if constexpr (QR == 32) {
            f32x16 acc = {};
#pragma unroll
            for (int st = 0; st < G::NS; ++st) {
                const f16x8 k8 = widen(x.k[st / 2][st % 2 * 2], x.k[st / 2][st % 2 * 2 + 1], ks0);
#pragma unroll
                for (int p = 0; p < PL; ++p) acc = mfma(k8, G::BIG ? query(p, st) : q[p][G::BIG ? 0 : st], acc);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = acc[i];
        } else {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < G::NS; ++st) {
                    const u32x4& w = x.k[kb * (G::KCH / 2) + st / 2];
                    const f16x8 k8 = widen(w[st % 2 * 2], w[st % 2 * 2 + 1], kb ? ks1 : ks0);
#pragma unroll
                    for (int p = 0; p < PL; ++p) acc = mfma(k8, G::BIG ? query(p, st) : q[p][G::BIG ? 0 : st], acc);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * kb + i] = acc[i];
            }
        }

        fetch_k(t + NW, x);

        // ---- masks: scores the row may not use
        uint32_t hidden = 0;
        const int key0 = 32 * t + G::NP * half;
        if (slow) {
            const u32x4 kw = gload<u32x4>(sbase + (size_t)t * 64 + (QR == 32 ? 16 * half : half / 2 * 16));
#pragma unroll
            for (int i = 0; i < G::NP; ++i) {
                const int key = key0 + i;
                const bool see = key < S.nk && visible(my_pos, key, 0, 0, a.window, a.prefix);
                const int kbyte = QR == 32 ? byte_of(kw, i)
                                           : (int)((half & 1 ? kw[2 + i / 4] : kw[i / 4]) >> (8 * (i % 4))) & 255;
                if (!see) {
                    hidden |= 1u << i;
                    s[i] = -INFINITY;
                } else if (kbyte == FP8_NAN) {
                    s[i] = NAN;
                }
            }
        }

        // ---- running maximum (moved rarely), probabilities, sum
        float top = s[0];
#pragma unroll
        for (int i = 1; i < G::NP; ++i) top = __builtin_fmaxf(top, s[i]);
        const float ts = top == -INFINITY ? -INFINITY : top * kc;
        if (__any(ts > m + MOVE)) {
            float nm = ts;
#pragma unroll
            for (int off = QR; off < 64; off <<= 1) nm = __builtin_fmaxf(nm, __shfl_xor(nm, off));
            nm = nm > m + MOVE ? nm : m;
            const float f = m == nm ? 1.0f : __builtin_amdgcn_exp2f(m - nm);
            m = nm;
            l *= f;
#pragma unroll
            for (int db = 0; db < G::DB; ++db) o[db] *= f;
        }
        const float off = P0 - (m == -INFINITY ? 0.0f : m);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        f16x8 vs[G::NP / 8];
#pragma unroll
        for (int i = 0; i < G::NP / 8; ++i) vs[i] = *reinterpret_cast<const f16x8*>(my_vs + G::NP * half + 8 * i);
        if (slow)  // (a hidden key's p is 0; a scale of infinity would still make it NaN)
#pragma unroll
            for (int i = 0; i < G::NP; ++i) vs[i / 8][i % 8] = hidden >> i & 1 ? (_Float16)0.0f : vs[i / 8][i % 8];
        f16x8 ph[G::NP / 8], pl[G::NP / 8];
#pragma unroll
        for (int i = 0; i < G::NP; i += 2) {
            const f32x2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], kc, off)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], kc, off))};
            const f16x2 hi = __builtin_convertvector(p, f16x2);
            if constexpr (PL == 1) {
                // the sum is of the weights that the product takes
                l = __builtin_amdgcn_fdot2(hi, f16x2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
            } else {
                l += p[0];
                l += p[1];
                const f32x2 r = {p[0] - (float)hi[0], p[1] - (float)hi[1]};
                const f16x2 lo = __builtin_convertvector(r, f16x2);
                pl[i / 8][i % 8] = lo[0];
                pl[i / 8][i % 8 + 1] = lo[1];
            }
            ph[i / 8][i % 8] = hi[0];
            ph[i / 8][i % 8 + 1] = hi[1];
        }
#pragma unroll
        for (int i = 0; i < G::NP / 8; ++i) {
            ph[i] *= vs[i];
            if constexpr (PL == 2) pl[i] *= vs[i];
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int db = 0; db < G::DB; ++db)
#pragma unroll
            for (int st = 0; st < G::NP / 8; ++st) {
                const f16x8 v8 = widen(x.v[(db * (G::NP / 8) + st) * 2], x.v[(db * (G::NP / 8) + st) * 2 + 1], 1.0f);
                o[db] = mfma(v8, ph[st], o[db]);
                if constexpr (PL == 2) o[db] = mfma(v8, pl[st], o[db]);
            }
        fetch_v(t + NW, x);
        // (the next tile's V scales are written after this tile's reads)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    for (int t = t_first; t < t1; t += NW) step(t, x);
    if constexpr (G::BIG) __syncthreads();  // (the merge area lies over the query rows)

    // ---- merge the waves
    float lt = l;
#pragma unroll
    for (int off = QR; off < 64; off <<= 1) lt += __shfl_xor(lt, off);
    if (half == 0) {
        sm[wave * QR + col] = m;
        sl[wave * QR + col] = lt;
    }
    __syncthreads();
    float M = sm[col];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = __builtin_fmaxf(M, sm[w * QR + col]);
    const float f = (m == -INFINITY ? (l != l ? l : 0.0f) : __builtin_amdgcn_exp2f(m - M)) * fp8_scale(vref);
    // (2^vref: the V scales' common factor)
#pragma unroll
    for (int db = 0; db < G::DB; ++db)
#pragma unroll
        for (int i = 0; i < G::SPL; i += 4) {
            // C layout: 4 consecutive O^T rows per four registers
            const int d = QR == 32 ? 32 * db + 2 * i + 4 * half : 16 * db + 4 * half;
            *reinterpret_cast<f32x4*>(so + (wave * QR + col) * G::OP + d) =
                f32x4{o[db][i] * f, o[db][i + 1] * f, o[db][i + 2] * f, o[db][i + 3] * f};
        }
    __syncthreads();
    // ---- this workgroup's rows: the sum relative to the row maximum M, and L
    constexpr int NT = NW * 64;
    const int nr = min(QR, rows - r0), items = nr * (HD / 4);
    auto state = [&](int i, int d, float& M, float& L) __attribute__((always_inline)) {
        M = sm[i];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = __builtin_fmaxf(M, sm[w * QR + i]);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = sm[w * QR + i], lw = sl[w * QR + i];
            L += mw == -INFINITY ? (lw != lw ? lw : 0.0f) : lw * __builtin_amdgcn_exp2f(mw - M);
            acc += *reinterpret_cast<const f32x4*>(so + (w * QR + i) * G::OP + d);
        }
        return acc;
    };
    if (a.n_split == 1) {
        for (int p = tid; p < items; p += NT) {
            const int i = p / (HD / 4), d = p % (HD / 4) * 4;
            float M, L;
            const f32x4 acc = state(i, d, M, L);
            write_out<HD>(a, S, g, r0 + i, d, acc * (1.0f / L));
        }
        return;
    }

    // ---- key splits.  Each workgroup stores its states with agent-scope
    // accesses and waits until they are complete; one thread then takes the row
    // block's ticket.  The one that draws n_split - 1 is the last: the others'
    // stores are complete and its agent-scope loads see them.  It joins the
    // splits in an order of its own (the same bits whichever comes last) and
    // resets the ticket for the next call.  No workgroup waits for another.
    // (Byte offsets of the workspace fit 32 bits: the host checks.)
    const size_t prow0 = ((size_t)b * a.n_head_kv + g) * a.part_rows + r0;
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.part_o, 0xffffffffu);
    const __amdgpu_buffer_rsrc_t rm = make_rsrc(a.part_ml, 0xffffffffu);
    for (int p = tid; p < items; p += NT) {
        const int i = p / (HD / 4), d = p % (HD / 4) * 4;
        float M, L;
        const f32x4 acc = state(i, d, M, L);
        const size_t at = (size_t)split * plane + prow0 + i;
        store_sc1(ro, (int)((at * HD + d) * 4), acc);
        // (a NaN without any finite score must not pass for a row without keys)
        if (d == 0) store2_sc1(rm, (int)(at * 8), L != L && M == -INFINITY ? 0.0f : M, L);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* const tk = a.ticket + (b * a.n_head_kv + g) * a.rowgroups + rb;
    if (tid == 0) *stick = __hip_atomic_fetch_add(tk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*stick != a.n_split - 1) return;
    if (tid == 0) __hip_atomic_store(tk, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Few rows leave threads over: `share` threads take an item's splits (thread
    // k of them takes splits k, k + share, ...), so that all loads of a wide split
    // are in flight together; their states join through LDS.
    int share = 1;
    while (2 * share * items <= NT) share *= 2;
    float* const sj = so;  // [share][items][6]
    for (int p = tid; p < share * items; p += NT) {
        const int k = p / items, it = p - k * items, i = it / (HD / 4), d = it % (HD / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int s0 = k; s0 < a.n_split; s0 += 8 * share) {
            float m[8], l[8];
            f32x4 o8[8][1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int sp = s0 + j * share;
                const size_t at = (size_t)min(sp, a.n_split - 1) * plane + prow0 + i;
                const float2 ml = load2_sc1(rm, (int)(at * 8));
                o8[j][0] = load_sc1(ro, (int)((at * HD + d) * 4));
                m[j] = sp < a.n_split ? ml.x : -INFINITY;
                l[j] = ml.y;
            }
            __builtin_amdgcn_sched_barrier(0);  // (every load above before any wait)
            merge_split_states<8, 1>(M, L, acc, m, l, o8);
        }
        if (share == 1) {
            write_out<HD>(a, S, g, r0 + i, d, acc[0] * (1.0f / L));
        } else {
            float* t = sj + p * 6;
            t[0] = M;
            t[1] = L;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[2 + e] = acc[0][e];
        }
    }
    if (share == 1) return;
    __syncthreads();
    if (tid < items) {
        float M = -INFINITY, L = 0.0f;
        f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int k = 0; k < share; ++k) {
            const float* t = sj + (k * items + tid) * 6;
            const float m[1] = {t[0]}, l[1] = {t[1]};
            const f32x4 w[1][1] = {{{t[2], t[3], t[4], t[5]}}};
            merge_split_states<1, 1>(M, L, acc, m, l, w);
        }
        write_out<HD>(a, S, g, r0 + tid / (HD / 4), tid % (HD / 4) * 4, acc[0] * (1.0f / L));
    }
}

template <int HD, int QR, int PL, int NW>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
    using G = Fp8Geo<HD, QR, PL, NW>;
    static_assert(G::LDS <= 160 * 1024, "LDS");
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_fp8_kernel<HD, QR, PL, NW>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::LDS);
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)((a.n_wg + 7) / 8 * 8));
    hipLaunchKernelGGL((attn_fp8_kernel<HD, QR, PL, NW>), grid, dim3(NW * 64), G::LDS, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_hd(const LaunchPlan& p, const AttnArgs& a, hipStream_t st) {
    const bool one = a.q_bf16 && a.o_bf16;
    hipError_t e = hipErrorInvalidValue;
    if constexpr (HD <= 128) {
        if (p.w16)
            e = p.waves == 8 ? (one ? launch<HD, 16, 1, 8>(a, st) : launch<HD, 16, 2, 8>(a, st))
                             : (one ? launch<HD, 16, 1, 4>(a, st) : launch<HD, 16, 2, 4>(a, st));
        else
            e = p.waves == 8 ? (one ? launch<HD, 32, 1, 8>(a, st) : launch<HD, 32, 2, 8>(a, st))
                             : (one ? launch<HD, 32, 1, 4>(a, st) : launch<HD, 32, 2, 4>(a, st));
    } else if (p.w16 && p.waves == 4) {
        e = one ? launch<HD, 16, 1, 4>(a, st) : launch<HD, 16, 2, 4>(a, st);
    }
    return e;
}

}  // namespace

LaunchPlan plan_fp8(int hd_tile, int n_batch, int n_head_kv, int group, int max_nq, int max_nk, int mask, int n_cu,
                    int force_split, int max_tickets) {
    LaunchPlan p{};
    p.hd_tile = hd_tile;
    p.block_n = 32;
    p.rb = 1;
    p.kq = 1;
    p.stages = 1;
    p.mask = mask;
    p.kernel = KERNEL_FP8;
    p.w16 = hd_tile > 128 || group * max_nq <= 16;
    const int qr = p.w16 ? 16 : 32;
    p.rowgroups = (group * max_nq + qr - 1) / qr;
    const int base = n_batch * n_head_kv * p.rowgroups;
    const int tiles = std::max(1, (max_nk + 31) / 32);
    // 8 waves where a workgroup per CU is all there is, else 4 (two workgroups per CU)
    p.waves = hd_tile <= 128 && base <= n_cu ? 8 : 4;
    const int slots = p.waves == 8 ? n_cu : 2 * n_cu;
    int split = 1;
    if (force_split > 0)
        split = force_split;
    else if (2 * base <= slots)
        split = std::min(slots / base, (tiles + p.waves - 1) / p.waves);
    p.n_split = std::max(1, split);
    // (the splits' tickets, and 32-bit offsets into their workspace: only a
    // forced split can outgrow them)
    if (base > max_tickets || split_workspace_bytes(p, n_batch, n_head_kv) >= ((size_t)1 << 31)) p.n_split = 1;
    p.n_workgroups = base * p.n_split;
    return p;
}

hipError_t launch_fp8(const LaunchPlan& p, const AttnArgs& a, hipStream_t st) {
    switch (p.hd_tile) {
        case 64: return launch_hd<64>(p, a, st);
        case 128: return launch_hd<128>(p, a, st);
        case 256: return launch_hd<256>(p, a, st);
        case 512: return launch_hd<512>(p, a, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dr
