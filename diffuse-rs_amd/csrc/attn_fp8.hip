// attn_fp8.hip -- attention over a DR_PRECISION_FP8 cache layer (arithmetic:
// fp8_attn.hpp).
//
// A workgroup owns QR packed rows of one KV head (row r = query * group + head
// in group, so a block spans few positions) and a range of 32-key tiles; its NW
// waves take tiles t, t + NW, ..., each with its own state, and merge through
// LDS.  Tiles come straight from memory into registers: the planes hold a tile
// in operand order, so every load is one contiguous run.  A step refills K's
// registers once its scores are formed and V's once its product is, so the
// loads run under the rest of the step and a tile ahead costs no registers.
// Few workgroups split the keys further; the last of a row block to finish
// joins them.
//
// What bounds it.  One row over a long cache: the stream of the codes (f32 row,
// 32/8 heads of 128, 131072 keys: 268 MB in 53 us, 5.0 TB/s, where a copy reaches
// 5.2).  Few tiles: latencies in a row, arguments 1 us, query rows 1, first tiles
// 2-4, the waves' meeting 2 (256 f32 rows, 32 heads, 768 keys: 12-13 us, of which
// 5.5 are the products' and 4 the bytes').  Many tiles: the vector units, 233
// instructions a tile and wave at 4.3-6.6 clk beside 16 or 32 MFMAs of 32 (4096
// bf16 rows, 32 heads, causal: 138 GFLOP in 200 us, 690 TFLOP/s; counters: vector
// units 61 %, matrix cores 29 % of the time, which nearly add up).  f32 rows at
// head dim 256 spill 23 registers (256 rows, 16/8 heads, window 1024: 19.2 us,
// bf16 rows 17.5).  Tried
// there without gain: three waves a SIMD (199 against 200 us), 64 rows a wave so
// that codes are widened once for two blocks (265, registers), tiles shared
// through LDS (255-290), waves on different rows (215-222).
#include "fp8_attn.hpp"

#include <algorithm>
#include <cmath>

namespace dr {
namespace {

template <int HD, int QR, int PL, int NW>
struct Fp8Geo {
    static constexpr int KCH = HD * 32 / 16 / 64;     // 16-byte K pieces per lane and tile
    static constexpr int VW = HD * 32 / 4 / 64;       // dwords of V per lane and tile
    // Head dim 512: the query planes (128 registers) are read from LDS as they
    // are multiplied, for the registers' sake.
    static constexpr bool BIG = HD > 256;
    static constexpr int QP = HD + 8;                 // f16 pitch of a staged query row
    static constexpr size_t Q_BYTES = (size_t)PL * QR * QP * 2;
    static constexpr size_t O_BYTES = (size_t)NW * QR * (HD + 4) * 4;
    static constexpr size_t BODY = O_BYTES > Q_BYTES ? O_BYTES : Q_BYTES;
    // then: per-row scales, wave states, row states, V scales (f16) of each wave's tile, the ticket
    static constexpr size_t LDS = BODY + QR * 4 + 2 * NW * QR * 4 + 2 * QR * 4 + NW * 32 * 2 + 16;
};

template <int HD, int QR, int PL, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(HD > 256 ? 1 : 2)))
void attn_fp8_kernel(const AttnArgs a) {
    using G = Fp8Geo<HD, QR, PL, NW>;
    using T = Fp8State<HD, QR, PL>;
    extern __shared__ __align__(16) char lds[];
    _Float16* const sq = reinterpret_cast<_Float16*>(lds);  // [PL][QR][QP]
    int* const srow = reinterpret_cast<int*>(lds + G::BODY);
    float* const sm = reinterpret_cast<float*>(srow + QR);
    float* const sl = sm + NW * QR;
    float* const sr = sl + NW * QR;
    _Float16* const svs = reinterpret_cast<_Float16*>(sr + 2 * QR);  // [NW][32]
    int* const stick = reinterpret_cast<int*>(svs + NW * 32);

    AttnSlot S = request_args(a);
    const Fp8Place at(a);
    if (!at.ok) return;
    if (a.n_batch > 1) S = a.slot[at.b];
    const int rows = S.nq * a.group, r0 = at.rg * QR;
    if (r0 >= rows) return;  // (a shorter pass of the batch)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane % QR, half = lane / QR;  // query column; 0..1 (0..3 with 16 rows)

    Fp8Queries<HD, QR, PL, NW * 64, G::QP> queries;
    queries.load(a, S, at.g, r0, rows);

    // ---- the key tiles that this workgroup's rows can see
    const int q_lo = uniform_pos(S, udiv(r0, a.group, a.mg_group)), q_hi = uniform_pos(S, udiv(min(r0 + QR, rows) - 1, a.group, a.mg_group));
    const int my_pos = row_pos(S, udiv(min(r0 + col, rows - 1), a.group, a.mg_group));
    int kt_lo, kt_hi, t0, t1;
    row_tiles(a, S.nk, q_lo, q_hi, kt_lo, kt_hi);
    split_tile_range(kt_lo, kt_hi, a.n_split, at.split, t0, t1);

    const uint8_t* const kbase = reinterpret_cast<const uint8_t*>(S.k) + fp8_tile(at.g, a.cap, 0, HD);
    const uint8_t* const vbase = reinterpret_cast<const uint8_t*>(S.vt) + fp8_tile(at.g, a.cap, 0, HD);
    const uint8_t* const sbase = reinterpret_cast<const uint8_t*>(S.klo) + fp8_scale_tile(at.g, a.cap, 0);
    const int last_tile = a.cap / 32 - 1;

    struct Tile {
        u32x4 k[G::KCH];
        uint32_t v[G::VW];
        int kb0, kb1, vb;  // scale bytes: K's of this lane's A rows, V's of key lane % 32
    };
    // (a tile past the plane's end, which nobody multiplies, is its last one)
    auto fetch_k = [&](int t, Tile& x) __attribute__((always_inline)) {
        t = min(t, last_tile);
        const uint8_t* kt = kbase + (size_t)t * 32 * HD;
        const uint8_t* st = sbase + (size_t)t * 64;
        x.vb = gload<uint8_t>(st + 32 + (lane & 31));
        if constexpr (QR == 32) {
            const int key = sigma(col);
            x.kb0 = x.kb1 = gload<uint8_t>(st + key);
#pragma unroll
            for (int j = 0; j < G::KCH; ++j) x.k[j] = gload<u32x4>(kt + (2 * j + half) * 512 + key * 16);
        } else {
            x.kb0 = gload<uint8_t>(st + kappa(col));
            x.kb1 = gload<uint8_t>(st + kappa(16 + col));
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
            for (int db = 0; db < T::DB; ++db) {
                const u32x4 w = gload<u32x4>(vt + (32 * db + col) * 32 + half * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.v[4 * db + e] = w[e];
            }
        } else {
#pragma unroll
            for (int db = 0; db < T::DB; ++db) {
                const u32x2 w = gload<u32x2>(vt + (16 * db + col) * 32 + half * 8);
                x.v[2 * db] = w[0];
                x.v[2 * db + 1] = w[1];
            }
        }
    };

    Tile x;
    const int t_first = t0 + wave;
    if (t_first < t1) {  // (in flight behind the query rows while those are staged)
        fetch_k(t_first, x);
        fetch_v(t_first, x);
    }
    queries.stage(a, sq, srow);
    __syncthreads();
    auto staged = [&](int p, int s) __attribute__((always_inline)) {
        // K piece j of a lane holds 16 values, steps 2j and 2j + 1
        const int d = ((64 / QR) * (s / 2) + half) * 16 + s % 2 * 8;
        return *reinterpret_cast<const f16x8*>(sq + (p * QR + col) * G::QP + d);
    };
    f16x8 q[PL][G::BIG ? 1 : T::NS];
    if constexpr (!G::BIG)
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int s = 0; s < T::NS; ++s) q[p][s] = staged(p, s);

    T st;
    auto walk = [&](auto far) __attribute__((always_inline)) {
        st.init(a.c, srow[col]);
        for (int t = t_first, cap = FP8_NAN; t < t1;) {
            int then = t;
            const int next = st.template tile<decltype(far)::value>(
                cap, x.kb0, x.kb1, x.vb, svs + wave * 32, !tile_visible(a, S.nk, t, q_lo, q_hi),
                [&](int kb, int s) {
                    const u32x4& w = x.k[kb * (G::KCH / 2) + s / 2];
                    return u32x2{w[s % 2 * 2], w[s % 2 * 2 + 1]};
                },
                [&](int db, int s) {
                    const int i = (db * (T::NP / 8) + s) * 2;
                    return u32x2{x.v[i], x.v[i + 1]};
                },
                [&](int p, int s) { return G::BIG ? staged(p, s) : q[p][G::BIG ? 0 : s]; },
                [&](int i) {
                    const int key = 32 * t + T::NP * half + i;
                    return (key < S.nk) & visible(my_pos, key, 0, 0, a.window, a.prefix);
                },
                [&](int i) { return (int)gload<uint8_t>(sbase + (size_t)t * 64 + T::NP * half + i); },
                [&](int again) {
                    then = again ? t : t + NW;
                    fetch_k(then, x);
                });
            fetch_v(then, x);
            t = then;
            cap = next ? next : FP8_NAN;
        }
    };
    walk(std::false_type{});
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(st.bad), 0)) {
        fetch_k(t_first, x);
        fetch_v(t_first, x);
        walk(std::true_type{});
    }
    if constexpr (G::BIG) __syncthreads();  // (the merge area lies over the query rows)
    fp8_finish<HD, QR, PL, NW>(a, S, at, st, r0, reinterpret_cast<float*>(lds), sm, sl, sr, stick);
}

template <int HD, int QR, int PL, int NW>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
    using G = Fp8Geo<HD, QR, PL, NW>;
    static_assert(G::LDS <= 160 * 1024, "LDS");
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_fp8_kernel<HD, QR, PL, NW>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_fp8_kernel<HD, QR, PL, NW>), dim3(fp8_grid(a)), dim3(NW * 64), G::LDS, st, a);
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
    } else if (!p.w16) {
        return HD > 256 ? launch_fp8_wide(a, st) : hipErrorInvalidValue;
    } else if (p.waves == 4) {
        e = one ? launch<HD, 16, 1, 4>(a, st) : launch<HD, 16, 2, 4>(a, st);
    }
    return e;
}

}  // namespace

// The launch shape of an 8 bit call.
//
// Row blocks: 16 rows where O^T of 32 would not fit the registers (head dims above
// 128) or where 16 hold all, else 32.  Head dims 257-512 with many rows take 64 in
// the wide kernel: it starts slower (24 us against 8 of fixed time) but a 32-key
// tile costs it 1.6 us for 64 rows, where four waves take 2.6 us for four tiles of
// 16 rows.  Measured, 16-row / wide, f32 rows over 2 KV heads of 512 dims, group 8:
// 256 rows (256 blocks) over 600 keys 25 / 38 us, 1800 49 / 54, 2800 68.5 / 69.2,
// 3200 75.5 / 74.8, 3800 88.8 / 83.6, 4352 98.6 / 92.3, 32768 680 / 531; 600 rows
// over 600 keys 69 / 48, over 4352 277 / 243.  So a block for each CU breaks even
// near 95 tiles; 120 keeps the 16-row kernel up to 6 % too long there.  (Few row
// blocks would be split often, and 64 rows are dear to join: 32 rows over 32768
// keys 117 / 147.)
//
// Waves: 8 where a workgroup per CU is all there is, else 4, two workgroups per CU.
// 8 / 4 waves: 256 f32 rows x 32 heads of 128 over 768 keys (256 workgroups) 13.8 /
// 14.7 us, 512 x 16 heads over 2553 29.0 / 32.1; 300 x 32/8 heads over 2000 (304)
// 40.4 / 34.2, 1000 bf16 rows (1000) 66 / 54.
//
// Key splits.  A step of a workgroup (one tile of each wave, or of the wide kernel)
// takes `step` us, a split's join reads its rows of floats at 13000 a us, and a join
// at all about 2 us: so steps / n * step + n * floats / 13000 is smallest at n =
// sqrt(steps * step * 13000 / floats).  More workgroups than CUs mostly wait for
// each other: 16 rows x 8 heads of 256 dims over 32768 keys (8 row blocks), 16 splits
// 38 us, 32 61; 1 / 2 / 3 splits of 160 row blocks, 160 rows x 32 heads of 128 over
// 4096 keys 30.7 / 42.6 / 35.8, 300 x 16 heads over 2553 22.7 / 34.5 / 28.4; of 200 at
// head dim 256, 4352 keys, 43.5 / 43.9 / 47.7.  (Not always: of 136 there, 130 rows,
// 43.5 / 41.8 / 33.7, and the rule does not split.)
// A split for every tile and CU, as cheap single rows take it, costs more rows up to
// twice the time (5 rows x 16/2 heads of 512 dims, 4352 keys: 34 splits 44 us, 9 33).
LaunchPlan plan_fp8(int hd_tile, int n_batch, int n_head_kv, int group, int max_nq, int max_nk, int mask, int n_cu,
                    int force_split, int force_rows, int max_tickets) {
    LaunchPlan p{};
    p.hd_tile = hd_tile;
    p.block_n = 32;
    p.stages = 1;
    p.mask = mask;
    p.kernel = KERNEL_FP8;
    const int tiles = std::max(1, (max_nk + 31) / 32), packed = group * max_nq;
    const int64_t base16 = (int64_t)n_batch * n_head_kv * ((packed + 15) / 16);
    const bool many = packed > 32 && (base16 > n_cu || (4 * base16 >= n_cu && base16 * tiles >= (int64_t)120 * n_cu));
    const bool wide = hd_tile > 256 && (force_rows ? force_rows == 32 : many);
    p.w16 = !wide && (hd_tile > 128 || (force_rows ? force_rows == 16 : packed <= 16));
    p.rb = wide ? 2 : 1;
    const int qr = p.w16 ? 16 : 32 * p.rb;
    p.rowgroups = (packed + qr - 1) / qr;
    const int base = n_batch * n_head_kv * p.rowgroups;
    p.waves = wide || (hd_tile <= 128 && base <= n_cu) ? 8 : 4;
    p.kq = wide ? 1 : p.waves;
    int split = 1;
    if (force_split > 0) {
        split = force_split;
    } else if (2 * base <= n_cu) {
        const float step = wide ? 1.6f : hd_tile > 256 ? 2.6f : p.w16 ? 1.0f : 1.3f;
        const int steps = (tiles + p.kq - 1) / p.kq;
        const float join = (float)(std::min(qr, packed) * hd_tile) / 13000.0f;
        split = std::clamp((int)std::sqrt((float)steps * step / join), 1, std::min(n_cu / base, steps));
        const int most = (steps + split - 1) / split;  // steps of a workgroup
        split = (steps + most - 1) / most;             // (no more splits than that takes)
        if ((float)(steps - most) * step < 2.0f + (float)split * join) split = 1;
    }
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
