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
#include "fp8_attn.hpp"

#include <algorithm>

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
    // scaled by a power of two each (inverse to srow), split into PL planes of f16
    // in sq [PL][QR][QP]
    __device__ __forceinline__ void stage(const AttnArgs& a, _Float16* sq, float* srow) const {
        const int tid = threadIdx.x, d0 = tid % LPR * 16;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int i = p * PER + tid / LPR;
            float up, down;
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

template <int HD, int QR, int PL, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(HD > 256 ? 1 : 2)))
void attn_fp8_kernel(const AttnArgs a) {
    using G = Fp8Geo<HD, QR, PL, NW>;
    using T = Fp8State<HD, QR, PL>;
    extern __shared__ __align__(16) char lds[];
    _Float16* const sq = reinterpret_cast<_Float16*>(lds);  // [PL][QR][QP]
    float* const srow = reinterpret_cast<float*>(lds + G::BODY);
    float* const sm = srow + QR;
    float* const sl = sm + NW * QR;
    float* const sr = sl + NW * QR;
    _Float16* const svs = reinterpret_cast<_Float16*>(sr + 2 * QR);  // [NW][32]
    int* const stick = reinterpret_cast<int*>(svs + NW * 32);

    const Fp8Place at(a);
    if (!at.ok) return;
    const AttnSlot& S = a.slot[at.b];
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
    st.init(fabsf(a.c) * srow[col]);
    for (int t = t_first; t < t1; t += NW) {
        st.tile(
            x.kb0, x.kb1, x.vb, svs + wave * 32, !tile_visible(a, S.nk, t, q_lo, q_hi),
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
            [&]() { fetch_k(t + NW, x); });
        fetch_v(t + NW, x);
    }
    if constexpr (G::BIG) __syncthreads();  // (the merge area lies over the query rows)
    fp8_finish<HD, QR, PL, NW>(a, at, st, r0, reinterpret_cast<float*>(lds), sm, sl, sr, stick);
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
    p.kq = p.waves;
    int split = 1;
    if (force_split > 0)
        split = force_split;
    else if (2 * base <= n_cu)
        split = std::min((p.waves == 8 ? 1 : 2) * n_cu / base, (tiles + p.waves - 1) / p.waves);
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
