// attn_fp8_wide.hip -- attention over a DR_PRECISION_FP8 cache layer at head dims
// 257-512 for many query rows (arithmetic: fp8_attn.hpp).
//
// A row block of 32 at head dim 512 needs 256 registers of O^T alone, so here a
// workgroup's 8 waves are two row blocks of 32 by four slices of the head dim:
// wave w holds Q and O^T of rows 32 (w / 4).. for dims 128 (w % 4).. and loads
// that slice of each tile.  A tile's scores are the sum of four waves' partial
// products: each writes its own to LDS, and after a barrier each sums a quarter of
// its block's scores (the keys 16 half + 4 (w % 4) .. + 3 of each lane half),
// turns them into weights and leaves those in LDS as the B operands that the four
// take for the values.  The values lag one tile behind the scores, so one barrier
// per tile orders both.  (Eight slices of 64 dims for both blocks widen every code
// once instead of twice, but put twice the partial scores and weights through
// LDS, which then bounds the loop.)
//
// The running maximum moves for the whole workgroup: a wave that meets a score
// more than 2^MOVE above it leaves the tile's number in LDS, and after the next
// barrier, before the weights are used, all waves exchange the row maxima,
// rescale and form the tile's weights again.
//
// What bounds it: 32 MFMAs of 32 clk a tile and wave are 2050 clk of a SIMD's
// 3400; the rest is the latency of LDS behind the barrier (104 KB a tile) and what
// of the weights no product covers.  256 f32 rows x 16/2 heads of 512 dims, 4352
// keys: 90-100 us, 36.5 GFLOP (twice that with both planes), of which starting is
// 9 us and joining the 4 splits 13.  Two planes spill 7 registers.
#include "fp8_attn.hpp"

namespace dr {
namespace {

template <int PL>
struct WideGeo {
    static constexpr int HD = 512, NW = 8, RB = 2, DW = HD / 4, ROWS = 32 * RB;
    static constexpr int QP = HD + 8;                  // f16 pitch of a staged query row
    static constexpr int PART = NW * 4096;        // a tile's partial scores
    static constexpr int PBUF = RB * PL * 2048;        // a tile's weights
    static constexpr size_t OUT = (size_t)ROWS * (HD + 4) * 4, QUERY = (size_t)PL * ROWS * QP * 2;
    // (the staged query rows and the rows of O lie over the tiles' buffers, both doubled)
    static constexpr size_t BODY = std::max({(size_t)2 * (PART + PBUF), OUT, QUERY});
    // then: row scales, row maxima of each wave, sums of each wave, two tile numbers, the ticket
    static constexpr size_t LDS = BODY + ROWS * 4 + NW * 32 * 4 * 2 + 16 + 16;
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int PL>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void attn_fp8_wide_kernel(const AttnArgs a) {
    using G = WideGeo<PL>;
    constexpr int HD = G::HD, NW = G::NW, NS = G::DW / 16, DB = G::DW / 32;
    extern __shared__ __align__(16) char lds[];
    char* const part = lds;
    char* const pbuf = lds + 2 * G::PART;
    int* const srow = reinterpret_cast<int*>(lds + G::BODY);          // [ROWS]
    float* const smax = reinterpret_cast<float*>(srow + G::ROWS);  // [NW][32]
    float* const ssum = smax + NW * 32;                           // [NW][32]
    int* const sflag = reinterpret_cast<int*>(ssum + NW * 32);    // [2]
    int* const stick = sflag + 4;

    AttnSlot S = request_args(a);
    const Fp8Place at(a);
    if (!at.ok) return;
    if (a.n_batch > 1) S = a.slot[at.b];
    const int rows = S.nq * a.group, r0 = at.rg * G::ROWS;
    if (r0 >= rows) return;  // (a shorter pass of the batch)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, half = lane >> 5;
    // this wave's row block and slice; it sums the scores of keys 16 half + 4 quad + j
    const int rb = wave >> 2, quad = wave & 3;

    const int q_lo = uniform_pos(S, udiv(r0, a.group, a.mg_group));
    const int q_hi = uniform_pos(S, udiv(min(r0 + G::ROWS, rows) - 1, a.group, a.mg_group));
    const int my_pos = row_pos(S, udiv(min(r0 + 32 * rb + col, rows - 1), a.group, a.mg_group));
    const int nk = S.nk;
    int kt_lo, kt_hi, t0, t1;
    row_tiles(a, nk, q_lo, q_hi, kt_lo, kt_hi);
    split_tile_range(kt_lo, kt_hi, a.n_split, at.split, t0, t1);

    const uint8_t* const kbase = reinterpret_cast<const uint8_t*>(S.k) + fp8_tile(at.g, a.cap, 0, HD);
    const uint8_t* const vbase = reinterpret_cast<const uint8_t*>(S.vt) + fp8_tile(at.g, a.cap, 0, HD);
    const uint8_t* const sbase = reinterpret_cast<const uint8_t*>(S.klo) + fp8_scale_tile(at.g, a.cap, 0);
    const int last_tile = a.cap / 32 - 1, key = sigma(col);

    // This wave's slice of a tile: K pieces of dims 128 quad + 32 j + 16 half, V rows
    // of dims 128 quad + 32 db + col; the scale bytes of K's row and of V's key col,
    // and V's of the four keys that this lane sums.
    struct Scales {
        int kb, vb;
        uint32_t vq;
    };
    auto fetch_k = [&](int t, Scales& x, u32x4 (&k)[DB]) __attribute__((always_inline)) {
        t = min(t, last_tile);  // (a tile past the plane's end, which nobody multiplies, is its last one)
        const uint8_t* kt = kbase + (size_t)t * 32 * HD + quad * G::DW * 32;
        const uint8_t* st = sbase + (size_t)t * 64;
        x.kb = gload<uint8_t>(st + key);
        x.vb = gload<uint8_t>(st + 32 + col);
        x.vq = gload<uint32_t>(st + 32 + 16 * half + 4 * quad);
#pragma unroll
        for (int j = 0; j < DB; ++j) k[j] = gload<u32x4>(kt + (2 * j + half) * 512 + key * 16);
    };
    auto fetch_v = [&](int t, u32x4 (&v)[DB]) __attribute__((always_inline)) {
        const uint8_t* vt = vbase + (size_t)t * 32 * HD + quad * G::DW * 32;
#pragma unroll
        for (int db = 0; db < DB; ++db) v[db] = gload<u32x4>(vt + (32 * db + col) * 32 + half * 16);
    };

    Fp8Queries<HD, G::ROWS, PL, 512, G::QP> queries;
    queries.load(a, S, at.g, r0, rows);
    queries.stage(a, reinterpret_cast<_Float16*>(lds), srow);
    if (tid < 2) sflag[tid] = 0;
    __syncthreads();
    f16x8 q[PL][NS];
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = quad * G::DW + s / 2 * 32 + half * 16 + s % 2 * 8;
            q[p][s] = *reinterpret_cast<const f16x8*>(reinterpret_cast<_Float16*>(lds) +
                                                      ((size_t)p * G::ROWS + rb * 32 + col) * G::QP + d);
        }
    const int eq = srow[32 * rb + col];
    __syncthreads();  // (the partial scores lie over the query rows)

    f32x16 o[DB];
    float m, l;         // row col's maximum; this lane's part of its sum
    int kref, vref, vfirst;  // (as of Fp8State)
    bool apart = false, bad = false;
    float kc;
    auto init = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
        kref = vref = vfirst = 0;
        kc = FLT_MIN;
    };
    init();
    // the tile whose weights wait in LDS: its scores and what turns them into weights
    float s[4], s_kc = 0.0f, l_before = 0.0f;
    f16x2 s_vs[2];

    // weights exp2(kept scores + off) into buffer b
    auto weigh = [&](int b, float off) __attribute__((always_inline)) {
        l = l_before;
        char* const to = pbuf + b * G::PBUF + rb * PL * 2048 + (quad >> 1) * 1024 + lane * 16 + (quad & 1) * 8;
        f16x2 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const f32x2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], s_kc, off)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e + 1], s_kc, off))};
            hi[e] = __builtin_convertvector(p, f16x2);
            if constexpr (PL == 1) {
                l = __builtin_amdgcn_fdot2(hi[e], f16x2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
            } else {
                l += p[0];
                l += p[1];
                lo[e] = __builtin_convertvector(residual(p, hi[e]), f16x2) * s_vs[e];
            }
            hi[e] *= s_vs[e];
        }
        *reinterpret_cast<u32x2*>(to) = u32x2{__builtin_bit_cast(uint32_t, hi[0]), __builtin_bit_cast(uint32_t, hi[1])};
        if constexpr (PL == 2)
            *reinterpret_cast<u32x2*>(to + 2048) =
                u32x2{__builtin_bit_cast(uint32_t, lo[0]), __builtin_bit_cast(uint32_t, lo[1])};
    };

    // tile k's weights (buffer k & 1) as B operands, and the tile number beside them
    auto weights = [&](int k, f16x8 (&w)[2][PL]) __attribute__((always_inline)) {
        const char* const from = pbuf + (k & 1) * G::PBUF + rb * PL * 2048 + lane * 16;
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int p = 0; p < PL; ++p) w[st][p] = *reinterpret_cast<const f16x8*>(from + (p * 2 + st) * 1024);
    };
    // Whether tile k's weights hold; else they are formed and read again.
    auto settle = [&](int k, int flag, f16x8 (&w)[2][PL]) __attribute__((always_inline)) {
        if (__builtin_amdgcn_readfirstlane(flag) == k + 1) {
            // some score was too far above its row's maximum
            float top = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
            top = top == -INFINITY ? -INFINITY : top * s_kc;
            top = __builtin_fmaxf(top, __shfl_xor(top, 32));
            if (half == 0) smax[wave * 32 + col] = top;
            lds_barrier();
            float nm = smax[rb * 128 + col];
#pragma unroll
            for (int w = 1; w < 4; ++w) nm = __builtin_fmaxf(nm, smax[(rb * 4 + w) * 32 + col]);
            nm = nm > m + MOVE ? nm : m;
            const float f = m == nm ? 1.0f : __builtin_amdgcn_exp2f(m - nm);
            m = nm;
            l_before *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= f;
            weigh(k & 1, P0 - (m == -INFINITY ? 0.0f : m));
            lds_barrier();
            weights(k, w);
        }
    };
    // a tile's values
    auto values = [&](const f16x8 (&w)[2][PL], const u32x4 (&v)[DB]) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const f16x8 v8 = widen(v[db][2 * st], v[db][2 * st + 1], 1.0f);
#pragma unroll
                for (int p = 0; p < PL; ++p) o[db] = mfma(v8, w[st][p], o[db]);
            }
        }
    };

    Scales x;
    u32x4 kq[DB], vq[DB];
    // Walk k of this workgroup: tile t's scores, the values of the walk before, its
    // weights.  (cap and t as of Fp8State::tile and its loop.)
    int t = t0, cap = FP8_NAN;
    auto step = [&](auto far_way, int k) __attribute__((always_inline)) {
        constexpr bool FAR = decltype(far_way)::value;
        // ---- K's and V's scales, the partial scores
        bool nan = false;
        float vdown = 1.0f;
        int next = 0;
        Band band{};
        bool banded = FAR && cap != FP8_NAN;
        if (__any((unsigned)(x.kb - kref + TK) > (unsigned)TK || (unsigned)(x.vb - vref + TV<PL>) > (unsigned)TV<PL> ||
                  (FAR && (apart || banded)))) {
            // (the same decisions in every wave: each sees all 64 bytes)
            const int k0 = x.kb > min(cap, FP8_NAN - 1) ? 0 : x.kb;
            const int kt = wave_max(k0), vt = wave_max(x.vb == FP8_NAN ? 0 : x.vb);
            nan = __any(x.kb == FP8_NAN || x.vb == FP8_NAN);
            if (kt > kref || __any(scale_far(k0, kref, TK)) || (FAR && kt > 0)) {
                kref = kt;
                kc = __builtin_fmaxf(ldexpf(fabsf(a.c), eq + kref - 127 - 7), FLT_MIN);
            }
            const bool steep = vfirst > 0 && vt > vfirst + TV_RISE;
            if constexpr (FAR) {
                next = wave_max(scale_far(k0, kref, TK) ? k0 : 0);
                banded = banded || next > 0;
                band = {kref, cap == FP8_NAN, next == 0};
            } else if (__builtin_expect(__any(scale_far(k0, kref, TK) || scale_far(x.vb, max(vref, vt), TV<PL>)) ||
                                            steep, 0)) {
                bad = true;
            }
            if (!(FAR && apart) && vt > vref && !steep) {
                if (vref > 0)
                    vdown = pow2_biased(vref - vt + 127);
                else
                    vfirst = vt;
                vref = vt;
            }
            if constexpr (FAR) apart = apart || __any(scale_far(x.vb, vref, TV<PL>));
        }
        const bool far = FAR && __builtin_amdgcn_readfirstlane(apart);
        const bool slow = __builtin_amdgcn_readfirstlane(!tile_visible(a, nk, t, q_lo, q_hi));
        const uint32_t vbytes = x.vq;
        f16x2 vs[2];  // V's scales of the four keys
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int vb = (int)(vbytes >> (8 * j)) & 255;
            vs[j / 2][j % 2] = (_Float16)(vb == FP8_NAN ? INFINITY : pow2_biased(vb - vref + 127));
        }
        f32x16 acc = {};
        const float ks = band_scale(x.kb, kref);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const u32x4& w = kq[st / 2];
            const f16x8 k8 = widen(w[st % 2 * 2], w[st % 2 * 2 + 1], ks);
#pragma unroll
            for (int p = 0; p < PL; ++p) acc = mfma(k8, q[p][st], acc);
        }
        if constexpr (FAR) next = __builtin_amdgcn_readfirstlane(next);
        const int then = next ? t : t + 1;
        fetch_k(then, x, kq);
        char* const mine = part + (k & 1) * G::PART + wave * 4096 + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(mine + i * 1024) = f32x4{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
        lds_barrier();

        // what this wave takes from LDS, in one go
        const char* const from = part + (k & 1) * G::PART + rb * 4 * 4096 + quad * 1024 + lane * 16;
        f32x4 pr[4];
        f16x8 w[2][PL];
#pragma unroll
        for (int w4 = 0; w4 < 4; ++w4) pr[w4] = *reinterpret_cast<const f32x4*>(from + w4 * 4096);
        const int flag = sflag[(k + 1) & 1];
        weights(k + 1, w);  // (tile k - 1's buffer)
        __builtin_amdgcn_sched_barrier(0);
        // this wave's scores, and their weights
        auto masked = [&]() __attribute__((always_inline)) {
            f32x4 sum = pr[0];
#pragma unroll
            for (int w = 1; w < 4; ++w) sum += pr[w];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = sum[j];
            s_vs[0] = vs[0];
            s_vs[1] = vs[1];
            s_kc = kc;
            if (FAR && banded) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!band.holds(gload<uint8_t>(sbase + (size_t)t * 64 + 16 * half + 4 * quad + j))) {
                        s[j] = -INFINITY;
                        s_vs[j / 2][j % 2] = (_Float16)0.0f;
                    }
            }
            if (nan)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (gload<uint8_t>(sbase + (size_t)t * 64 + 16 * half + 4 * quad + j) == FP8_NAN && s[j] != -INFINITY)
                        s[j] = NAN;
            if (slow)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int kk = 32 * t + 16 * half + 4 * quad + j;
                    if (!((kk < nk) & visible(my_pos, kk, 0, 0, a.window, a.prefix))) {
                        s[j] = -INFINITY;
                        s_vs[j / 2][j % 2] = (_Float16)0.0f;  // (0 times a scale of infinity)
                    }
                }
        };
        auto scored = [&]() __attribute__((always_inline)) {
            masked();
            float top = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
            top = top == -INFINITY ? -INFINITY : top * kc;
            if (__any(top > m + MOVE) && lane == 0) sflag[k & 1] = k + 1;
            l_before = l;
            weigh(k & 1, P0 - (m == -INFINITY ? 0.0f : m));
        };
        if (k > 0) settle(k - 1, flag, w);
        // Half of the waves, one of each SIMD's two, take the values of the tile
        // before first, the others their scores: the matrix cores and the vector
        // units both have work at any time.
        if (wave >= 4 && !far) scored();
        if (k > 0) values(w, vq);
        fetch_v(t, vq);
        if (__builtin_amdgcn_readfirstlane(__float_as_int(vdown)) != __float_as_int(1.0f))
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= vdown;
        if (far) {
            // the row's accumulators at a size of their own, then its maximum, then
            // V's scales into the weights' exponents: each as all four waves see it
            auto row_most = [&](float* in, float x) __attribute__((always_inline)) {
                x = __builtin_fmaxf(x, __shfl_xor(x, 32));
                if (half == 0) in[wave * 32 + col] = x;
                lds_barrier();
#pragma unroll
                for (int w4 = 0; w4 < 4; ++w4) x = __builtin_fmaxf(x, in[(rb * 4 + w4) * 32 + col]);
                return x;
            };
            float big = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) big = __builtin_fmaxf(big, fabsf(o[db][i]));
            big = row_most(ssum, big);
            const int up = centre(big);
            vref = big == 0.0f ? 0 : vref - up;
            masked();
            float top = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
            float nm = row_most(smax, top == -INFINITY ? -INFINITY : top * kc);
            nm = nm > m + MOVE ? nm : m;
            const float f = m == nm ? 1.0f : __builtin_amdgcn_exp2f(m - nm), off = P0 - (nm == -INFINITY ? 0.0f : nm);
            m = nm;
            l *= f;
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int vb = (int)(vbytes >> (8 * j)) & 255;
                s[j] = __builtin_fmaf(s[j], kc, off);
                l += __builtin_amdgcn_exp2f(s[j]);
                if (vb != FP8_NAN) most = __builtin_fmaxf(most, s[j] + (float)(vb - vref));
            }
            most = row_most(ssum, most);
            const int rise = most > P0 + MOVE ? (int)__builtin_fminf(ceilf(most - P0), 252.0f) : 0;
            vref += rise;
            const int e = up - rise;
            const float f0 = pow2_biased(e / 2 + 127), f1 = pow2_biased(e - e / 2 + 127);
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = o[db] * f * f0 * f1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int vb = (int)(vbytes >> (8 * j)) & 255;
                s[j] = vb == FP8_NAN && s[j] != -INFINITY ? NAN : s[j] + (float)(vb - vref);
            }
            s_kc = 1.0f;
            s_vs[0] = s_vs[1] = f16x2{(_Float16)1.0f, (_Float16)1.0f};
            const float sum = l;
            weigh(k & 1, 0.0f);
            l = l_before = sum;
        } else if (wave < 4) {
            scored();
        }
        t = then;
        cap = next ? next : FP8_NAN;
    };

    if (t0 < t1) {
        fetch_k(t0, x, kq);
        int n = 0;
        while (t < t1) step(std::false_type{}, n++);
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(bad), 0)) {
            // scales too far apart for the common way: from the start, on the other
            // (all waves decide alike)
            lds_barrier();
            if (tid < 2) sflag[tid] = 0;
            lds_barrier();
            init();
            t = t0;
            fetch_k(t0, x, kq);
            n = 0;
            while (t < t1) step(std::true_type{}, n++);
        }
        lds_barrier();
        f16x8 w[2][PL];
        weights(n - 1, w);
        settle(n - 1, sflag[(n - 1) & 1], w);
        values(w, vq);
    }

    // ---- the rows' sums, and the rows, which leave through LDS: whole lines
    const float lt = l + __shfl_xor(l, 32);
    if (half == 0) ssum[wave * 32 + col] = lt;
    __syncthreads();
    constexpr int OP = HD + 4;
    float* const so = reinterpret_cast<float*>(lds);  // [ROWS][OP]
    const int nr = min(G::ROWS, rows - r0);
    const size_t prow0 = ((size_t)at.b * a.n_head_kv + at.g) * a.part_rows + r0;
    const size_t plane = (size_t)a.n_batch * a.n_head_kv * a.part_rows;
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.part_o, 0xffffffffu);
    const __amdgpu_buffer_rsrc_t rm = make_rsrc(a.part_ml, 0xffffffffu);
    // (split rows meet at 2^-LOW)
    const int e2 = vref - 127 - (a.n_split > 1 ? LOW : 0);
    const float up0 = pow2_biased(e2 / 2 + 127), up1 = pow2_biased(e2 - e2 / 2 + 127);
    const int i = rb * 32 + col;
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += ssum[(rb * 4 + w) * 32 + col];
    const float f = a.n_split == 1 ? 1.0f / L : 1.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<f32x4*>(so + i * OP + quad * G::DW + 32 * db + 2 * e + 4 * half) =
                f32x4{o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]} * f * up0 * up1;
    // (a NaN without any finite score must not pass for a row without keys)
    if (a.n_split > 1 && quad == 0 && half == 0 && i < nr)
        store2_sc1(rm, (int)(((size_t)at.split * plane + prow0 + i) * 8), L != L && m == -INFINITY ? 0.0f : m, L * pow2_biased(127 - LOW));
    __syncthreads();
    for (int p = tid; p < nr * (HD / 4); p += 512) {
        const int i = p / (HD / 4), d = p % (HD / 4) * 4;
        const f32x4 y = *reinterpret_cast<const f32x4*>(so + i * OP + d);
        if (a.n_split == 1)
            write_out<HD>(a, S, at.g, r0 + i, d, y);
        else
            store_sc1(ro, (int)((((size_t)at.split * plane + prow0 + i) * HD + d) * 4), y);
    }
    if (a.n_split > 1) fp8_join<HD, 512>(a, S, at, r0, nr, so, stick);
}

template <int PL>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
    using G = WideGeo<PL>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_fp8_wide_kernel<PL>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(attn_fp8_wide_kernel<PL>, dim3(fp8_grid(a)), dim3(512), G::LDS, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_wide(const AttnArgs& a, hipStream_t st) {
    return a.q_bf16 && a.o_bf16 ? launch<1>(a, st) : launch<2>(a, st);
}

}  // namespace dr
