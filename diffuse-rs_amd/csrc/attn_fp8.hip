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
// workgroups split the keys further; the partial states go to a workspace and
// fp8_merge_kernel joins them.
//
// A key that a row may not see never reaches its output: its p is set to 0 and
// its codes are finite always (a row that held a NaN has codes 0 and the NaN in
// its scale byte, which is applied to visible keys only).  A row that sees no
// key ends 0 * (1 / 0) = NaN, like the reference (attention.rs:181-185).
#include "attn_common.hpp"
#include "fp8_common.hpp"

#include <algorithm>
#include <type_traits>

#include <math.h>

namespace dr {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float P0 = 8.0f, MOVE = 7.0f;
constexpr int NW = 4;  // waves per workgroup

template <int HD, int QR, int PL>
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
    // are multiplied, and no tile is fetched ahead, for the registers' sake.
    static constexpr bool BIG = HD > 256;
    static constexpr int QP = HD + 8;                 // f16 pitch of a staged query row
    static constexpr int OP = HD + 4;                 // f32 pitch of a merged row
    static constexpr size_t Q_BYTES = (size_t)PL * QR * QP * 2;
    static constexpr size_t EPI_BYTES = (size_t)NW * HD * 4;
    static constexpr size_t O_BYTES = (size_t)NW * QR * OP * 4;
    static constexpr size_t BODY = O_BYTES > Q_BYTES + EPI_BYTES ? O_BYTES : Q_BYTES + EPI_BYTES;
    // then: per-row scales, wave states, V scales of each wave's tile
    static constexpr size_t LDS = BODY + QR * 4 + 2 * NW * QR * 4 + NW * 32 * 4;
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

// The query row of packed row r: its values with the Q epilogue applied
// (forward.rs:291-310: bias, RMSNorm with f32 squares summed in f64, RoPE), EPL
// consecutive ones per lane.  `scratch`: HD floats of this wave.
template <int HD>
__device__ __forceinline__ void load_query(const AttnArgs& a, const AttnSlot& S, int qi, int head, int pos,
                                           float* scratch, float (&y)[HD / 64]) {
#pragma clang fp contract(off)
    constexpr int EPL = HD / 64;
    const int lane = threadIdx.x & 63, d0 = lane * EPL, hd = a.hd;
    const size_t off = (size_t)qi * a.q_rstride + (size_t)head * hd + d0;
    if (a.q_bf16) {
        const uint16_t* q = static_cast<const uint16_t*>(S.q) + off;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            y[e] = d0 + e < hd ? __uint_as_float((uint32_t)gload<uint16_t>(q + e) << 16) : 0.0f;
    } else {
        const float* q = static_cast<const float*>(S.q) + off;
#pragma unroll
        for (int e = 0; e < EPL; ++e) y[e] = d0 + e < hd ? gload<float>(q + e) : 0.0f;
    }
    if (a.qb)
#pragma unroll
        for (int e = 0; e < EPL; ++e) y[e] += d0 + e < hd ? a.qb[(size_t)head * hd + d0 + e] : 0.0f;
    if (a.qn_w) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const float sq = y[e] * y[e];
            ss += (double)sq;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        const float sc = 1.0f / (float)sqrt(ss / (double)hd + (double)a.qn_eps);
#pragma unroll
        for (int e = 0; e < EPL; ++e) y[e] = y[e] * sc * (d0 + e < hd ? a.qn_w[d0 + e] : 0.0f);
    }
    if (a.rope) {
        const int half = a.rot / 2;
#pragma unroll
        for (int e = 0; e < EPL; ++e) scratch[d0 + e] = y[e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int d = d0 + e;
            if (d >= a.rot) continue;
            const int j = d < half ? d : d - half;
            const float2 t = *reinterpret_cast<const float2*>(a.rope + ((size_t)pos * half + j) * 2);
            y[e] = d < half ? rope_lo(y[e], scratch[d + half], t.x, t.y) : rope_hi(scratch[j], y[e], t.x, t.y);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

__device__ __forceinline__ int row_pos(const AttnSlot& S, int qi) { return S.qpos0 >= 0 ? S.qpos0 + qi : S.qpos[qi]; }

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

template <int HD, int QR, int PL>
__global__ __launch_bounds__(NW * 64) void attn_fp8_kernel(const AttnArgs a) {
    using G = Fp8Geo<HD, QR, PL>;
    using Acc = std::conditional_t<QR == 32, f32x16, f32x4>;
    extern __shared__ __align__(16) char lds[];
    _Float16* const sq = reinterpret_cast<_Float16*>(lds);                 // [PL][QR][QP]
    float* const sepi = reinterpret_cast<float*>(lds + G::Q_BYTES);        // [NW][HD]
    float* const so = reinterpret_cast<float*>(lds);                       // [NW][QR][OP], after the key loop
    float* const srow = reinterpret_cast<float*>(lds + G::BODY);           // [QR]
    float* const sm = srow + QR;                                           // [NW][QR]
    float* const sl = sm + NW * QR;                                        // [NW][QR]
    float* const svs = sl + NW * QR;                                       // [NW][32]

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
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int col = lane % QR, half = lane / QR;  // query column; 0..1 (0..3 with 16 rows)

    // ---- the query rows: scaled, split into planes, staged in LDS
    for (int i = wave; i < QR; i += NW) {
        float y[HD / 64];
        const int r = r0 + i;
        const bool ok = r < rows;
        const int rr = ok ? r : rows - 1, qi = rr / a.group;
        load_query<HD>(a, S, qi, g * a.group + rr - qi * a.group, a.rope ? row_pos(S, qi) : 0, sepi + wave * HD, y);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        // 2^14 <= |largest| * up < 2^15; a row with a NaN or an infinity gives NaN
        const int e = min(268 - (int)(top >> 23), 254);
        const float up = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : pow2_biased(e);
        if (lane == 0) srow[i] = pow2_biased(top >= 0x7f800000u ? 127 : 254 - e);
#pragma unroll
        for (int k = 0; k < HD / 64; ++k) {
            const float z = (a.c < 0.0f ? -y[k] : y[k]) * up;
            const _Float16 hi = (_Float16)z;
            sq[i * G::QP + lane * (HD / 64) + k] = hi;
            if constexpr (PL == 2) sq[(QR + i) * G::QP + lane * (HD / 64) + k] = (_Float16)(z - (float)hi);
        }
    }
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
    auto fetch = [&](int t, Tile& x) __attribute__((always_inline)) {
        t = min(t, last_tile);
        const uint8_t* kt = kbase + (size_t)t * 32 * HD;
        const uint8_t* vt = vbase + (size_t)t * 32 * HD;
        const uint8_t* st = sbase + (size_t)t * 64;
        if constexpr (QR == 32) {
            const int key = sigma(col);
#pragma unroll
            for (int j = 0; j < G::KCH; ++j) x.k[j] = gload<u32x4>(kt + (2 * j + half) * 512 + key * 16);
#pragma unroll
            for (int db = 0; db < G::DB; ++db) {
                const u32x4 w = gload<u32x4>(vt + (32 * db + col) * 32 + half * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.v[4 * db + e] = w[e];
            }
            x.kb = gload<uint8_t>(st + key);
        } else {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int key = kappa(16 * kb + col);
#pragma unroll
                for (int j = 0; j < G::KCH / 2; ++j)
                    x.k[kb * (G::KCH / 2) + j] = gload<u32x4>(kt + (4 * j + half) * 512 + key * 16);
            }
#pragma unroll
            for (int db = 0; db < G::DB; ++db) {
                const u32x2 w = gload<u32x2>(vt + (16 * db + col) * 32 + half * 8);
                x.v[2 * db] = w[0];
                x.v[2 * db + 1] = w[1];
            }
            x.kb = (int)gload<uint8_t>(st + kappa(col)) | (int)gload<uint8_t>(st + kappa(16 + col)) << 8;
        }
        x.vb = gload<uint8_t>(st + 32 + (lane & 31));
    };

    Acc o[G::DB];
#pragma unroll
    for (int db = 0; db < G::DB; ++db)
#pragma unroll
        for (int i = 0; i < G::SPL; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, l = 0.0f, kc = 0.0f;
    int kref = 0, vref = 0;
    float* const my_vs = svs + wave * 32;

    auto step = [&](int t, const Tile& x) __attribute__((always_inline)) {
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
            kc = ldexpf(cq, kref - 127 - 7);
            if (vt > vref) {
                const float f = pow2_biased(vref - vt + 127);
#pragma unroll
                for (int db = 0; db < G::DB; ++db) o[db] *= f;
                vref = vt;
            }
        }
        if (lane < 32) my_vs[lane] = x.vb == FP8_NAN ? INFINITY : pow2_biased(x.vb - vref + 127);
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
        const float off = P0 - m;
        float vs[G::NP];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < G::NP; i += 4) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(my_vs + G::NP * half + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) vs[i + e] = w[e];
        }
        f16x8 ph[G::NP / 8], pl[G::NP / 8];
#pragma unroll
        for (int i = 0; i < G::NP; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], kc, off));
            if (slow && (hidden >> i & 1)) p = 0.0f;
            l += p;
            float pv = p * vs[i];
            if (slow && (hidden >> i & 1)) pv = 0.0f;
            const _Float16 hi = (_Float16)pv;
            ph[i / 8][i % 8] = hi;
            if constexpr (PL == 2) pl[i / 8][i % 8] = (_Float16)(pv - (float)hi);
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
        // (the next tile's V scales are written after this tile's reads)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    const int t_first = t0 + wave;
    if (t_first < t1) {
        Tile x, y;
        if constexpr (G::BIG) {
            for (int t = t_first; t < t1; t += NW) {
                fetch(t, x);
                step(t, x);
            }
        } else {
        fetch(t_first, x);
        for (int t = t_first; t < t1; t += 2 * NW) {
            fetch(t + NW, y);
            step(t, x);
            if (t + NW >= t1) break;
            fetch(t + 2 * NW, x);
            step(t + NW, y);
        }
        }
    }
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
    const size_t prow0 = ((size_t)b * a.n_head_kv + g) * a.part_rows;
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    for (int p = tid; p < QR * (HD / 4); p += NW * 64) {
        const int i = p / (HD / 4), d = p % (HD / 4) * 4, r = r0 + i;
        if (r >= rows) continue;
        float Mr = sm[i];
#pragma unroll
        for (int w = 1; w < NW; ++w) Mr = __builtin_fmaxf(Mr, sm[w * QR + i]);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = sm[w * QR + i], lw = sl[w * QR + i];
            L += mw == -INFINITY ? (lw != lw ? lw : 0.0f) : lw * __builtin_amdgcn_exp2f(mw - Mr);
            acc += *reinterpret_cast<const f32x4*>(so + (w * QR + i) * G::OP + d);
        }
        if (a.n_split > 1) {
            const size_t at = (size_t)split * plane + prow0 + r;
            *reinterpret_cast<f32x4*>(a.part_o + at * HD + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(Mr, L);
        } else {
            write_out<HD>(a, S, g, r, d, acc * (1.0f / L));
        }
    }
}

// Joins the key splits: one thread per (packed row, four values).
template <int HD>
__global__ __launch_bounds__(256) void fp8_merge_kernel(const AttnArgs a) {
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    const size_t item = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= plane * (HD / 4)) return;
    const size_t prow = item / (HD / 4);
    const int d = (int)(item % (HD / 4)) * 4;
    const int bg = (int)(prow / a.part_rows), r = (int)(prow % a.part_rows);
    const int b = bg / a.n_head_kv, g = bg % a.n_head_kv;
    const AttnSlot& S = a.slot[b];
    if (r >= a.group * S.nq) return;
    float M = -INFINITY;
    for (int s = 0; s < a.n_split; ++s) M = __builtin_fmaxf(M, a.part_ml[((size_t)s * plane + prow) * 2]);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float L = 0.0f;
    for (int s = 0; s < a.n_split; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + ((size_t)s * plane + prow) * 2);
        const f32x4 w = *reinterpret_cast<const f32x4*>(a.part_o + ((size_t)s * plane + prow) * HD + d);
        const float f = ml.x == -INFINITY ? (ml.y != ml.y ? ml.y : 0.0f) : __builtin_amdgcn_exp2f(ml.x - M);
        L += f * ml.y;
        acc += w * f;
    }
    write_out<HD>(a, S, g, r, d, acc * (1.0f / L));
}

template <int HD, int QR, int PL>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
    using G = Fp8Geo<HD, QR, PL>;
    static_assert(G::LDS <= 160 * 1024, "LDS");
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_fp8_kernel<HD, QR, PL>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::LDS);
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)((a.n_wg + 7) / 8 * 8));
    hipLaunchKernelGGL((attn_fp8_kernel<HD, QR, PL>), grid, dim3(NW * 64), G::LDS, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_hd(const LaunchPlan& p, const AttnArgs& a, hipStream_t st) {
    const bool one = a.q_bf16 && a.o_bf16;
    hipError_t e;
    if constexpr (HD <= 128) {
        if (!p.w16)
            e = one ? launch<HD, 32, 1>(a, st) : launch<HD, 32, 2>(a, st);
        else
            e = one ? launch<HD, 16, 1>(a, st) : launch<HD, 16, 2>(a, st);
    } else {
        if (!p.w16) return hipErrorInvalidValue;
        e = one ? launch<HD, 16, 1>(a, st) : launch<HD, 16, 2>(a, st);
    }
    if (e != hipSuccess || p.n_split <= 1) return e;
    const size_t items = (size_t)a.n_batch * a.n_head_kv * a.part_rows * (HD / 4);
    hipLaunchKernelGGL(fp8_merge_kernel<HD>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

LaunchPlan plan_fp8(int hd_tile, int n_batch, int n_head_kv, int group, int max_nq, int max_nk, int mask, int n_cu,
                    int force_split) {
    LaunchPlan p{};
    p.hd_tile = hd_tile;
    p.block_n = 32;
    p.rb = 1;
    p.kq = 1;
    p.waves = NW;
    p.stages = 1;
    p.mask = mask;
    p.kernel = KERNEL_FP8;
    p.w16 = hd_tile > 128 || group * max_nq <= 16;
    const int qr = p.w16 ? 16 : 32;
    p.rowgroups = (group * max_nq + qr - 1) / qr;
    const int base = n_batch * n_head_kv * p.rowgroups;
    const int tiles = std::max(1, (max_nk + 31) / 32);
    int split = 1;
    if (force_split > 0)
        split = force_split;
    else if (2 * base <= 2 * n_cu)
        split = std::min(2 * n_cu / base, (tiles + NW - 1) / NW);
    p.n_split = std::max(1, split);
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
