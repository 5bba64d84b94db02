// mx_tile.hip -- products of E2M1 weights with microscaled activations, many
// rows: tiles staged through LDS, the block-scaled MFMA.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes, each
// 32 of a row scaled by a power of two: no value is unpacked.  Lane (r, g) =
// (lane % 16, lane / 16) holds of row r: 4 bit codes: block g (16 bytes); 8 bit
// codes: values 16 g .. 16 g + 15 and 64 more (the 16-byte pieces g and 4 + g of
// the 128); and block g's scale byte.  The weights are the A operand, so a lane's
// four sums are consecutive output columns of one activation row.
//
// A workgroup's tile goes over the columns in stages of SB * 128.  A stage's codes come by
// LDS DMA, 16 bytes a lane, STAGES - 1 stages ahead; columns behind a row's end and rows
// behind the last are out of the buffer's range and read as 0 codes.  Scale bytes come
// for 512 columns (a chunk) at a time, 16 bytes of a row (four bytes a row and 128
// columns were half of all requests to L2), and wait in registers, a lane's four bytes
// of a row in one, from which the MFMA takes the one it is told.  A wave issues its DMA
// between its products: all of it at the start of a stage, the address unit kept the
// products waiting.
//
// Gated, 8 bit activations: in two parts (mx_split), whose MFMAs bound it.
//
// 4096 rows through 4096 x 12288, bf16: 147-155 us (2.7 PFLOP/s); 2 x 12288 x 4096 gated 525-560 (twice
// 1.5 PFLOP/s; in one part 300, with 1 of 1000 codes on the other side of a border);
// 4 bit activations, 2553 rows through 18944 x 3584, 120-124.  The matrix instruction alone
// reaches 4.2 PFLOP/s on such codes (7.1 with 4 bit ones), at 2.0 GHz, which is what power
// leaves; a large library product of 8 bit numbers 2.9.  The matrix cores are busy 70 % of
// the CUs' cycles; the rest is the end of a tile (residuals and outputs, 15 us of the 150),
// lines that miss L2 (15 us) and the waves' meetings.  Measured and not kept: a meeting
// before a step's last products (same), lines asked for early into L2 (215 us: a wave's loads
// return in order), stores past the caches (163 us), tiles of 256 x 128, two a CU (174 us).
#include "mx_common.hpp"

namespace dr {
namespace {

// A workgroup of WM x WN waves, each with Q groups of 64 weight rows by TN tiles
// of 16 activation rows.  Group q of a wave is rows of `w` (gated: odd groups
// are rows of `up`, of the same output columns as the group before).  Tile i, row
// 4 g + e of a group is its weight row 16 g + 4 i + e, so that lane group g's sums
// over the four tiles are 16 consecutive output columns.
template <int AF_, bool GATED_, int WM_, int Q_, int WN_, int TN_, int SB_, int STAGES_>
struct TileGeom {
    static constexpr int AF = AF_, WM = WM_, Q = Q_, WN = WN_, TN = TN_, SB = SB_, STAGES = STAGES_;
    static constexpr bool GATED = GATED_, SPLIT = GATED && AF == MX_E4M3;  // (mx_split)
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GROUPS = WM * Q;                       // of 64 weight rows
    static constexpr int COLS = GROUPS * 64 / (GATED ? 2 : 1);  // output columns
    static constexpr int BN = WN * TN * 16;
    static constexpr int W_ROW = SB * 64, A_ROW = SB * (AF == MX_E4M3 ? 128 : 64);  // bytes of a row and stage
    static constexpr int W_BYTES = GROUPS * 64 * W_ROW, A_BYTES = BN * A_ROW;
    static constexpr int NW = W_BYTES / 1024, NA = A_BYTES / 1024;  // DMA instructions of a stage
    static constexpr int NSW = GROUPS, NSA = (BN + 63) / 64;        // of a chunk's scales
    static constexpr int NI_W = NW / WAVES, NI_A = NA / WAVES, NI = NI_W + NI_A;  // of a wave
    static constexpr int NI_S = (NSW + NSA + WAVES - 1) / WAVES;
    static constexpr int PARTS = 4 / SB;                           // stages of a chunk
    static constexpr int AHEAD = (STAGES - 1 + PARTS - 1) / PARTS;  // chunks that scales are asked for ahead
    static constexpr int STAGE = W_BYTES + A_BYTES, S_OFF = STAGE * STAGES, S_STAGE = NI_S * WAVES * 1024;
    static constexpr int LDS = S_OFF + (AHEAD + 1) * S_STAGE;
    static constexpr int FIT = 160 * 1024 / LDS * WAVES / 4;  // waves per SIMD that LDS leaves room for
    static constexpr int MOST = Q * TN >= 8 ? 2 : 4, PER_SIMD = FIT < 1 ? 1 : FIT < MOST ? FIT : MOST;
    static constexpr bool WHOLE = Q * 16 + TN * 8 <= 24;  // two steps' operands fit in registers
    static constexpr int BAND = AF == MX_E4M3 ? 8 : 4;
    static_assert(NW % WAVES == 0 && NA % WAVES == 0, "every wave issues the same number");
    static_assert(!GATED || Q % 2 == 0, "gate and up groups pair up in a wave");
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert((STAGES - 2) * NI < 64, "vmcnt");
};

// A wave's sums, 16-byte pieces (rows a multiple of 8, out and residual aligned): lane's
// activation rows tok1 + 16 j, columns c1 + 64 q .. + 15.  The residuals of all of them
// (f32: of half) are asked for before the first is used; lanes behind the last row or
// column read a valid place instead and write nothing.
template <bool BF16, int Q, int TN>
__device__ __forceinline__ void put_tile(const MxMatArgs& a, const f32x4m (&acc)[Q][4][TN], int tok1, int c1) {
    constexpr int JB = BF16 || TN < 2 ? TN : TN / 2, P = BF16 ? 2 : 4, E = 16 / P;  // pieces of 16 columns, their values
    constexpr size_t SIZE = BF16 ? 2 : 4;
    const char* const res = static_cast<const char*>(a.residual);
    char* const out = static_cast<char*>(a.out);
#pragma unroll
    for (int j0 = 0; j0 < TN; j0 += JB) {
        u32x4m y[JB][Q][P] = {};
        if (res) {
#pragma unroll
            for (int j = 0; j < JB; ++j)
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int h = 0; h < P; ++h)
                        y[j][q][h] = *reinterpret_cast<const u32x4m*>(
                            res + ((size_t)min(tok1 + (j0 + j) * 16, a.n - 1) * a.rows + min(c1 + q * 64 + h * E, a.rows - E)) * SIZE);
        }
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            const int tok = tok1 + (j0 + j) * 16;
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int h = 0; h < P; ++h) {
                    const int c0 = c1 + q * 64 + h * E;
                    u32x4m v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t b = y[j][q][h][e];
                        if constexpr (BF16)
                            v[e] = mx_bf16(acc[q][2 * h + e / 2][j0 + j][e % 2 * 2] + mx_f32(b & 0xffff)) |
                                   (uint32_t)mx_bf16(acc[q][2 * h + e / 2][j0 + j][e % 2 * 2 + 1] + __uint_as_float(b & 0xffff0000u)) << 16;
                        else
                            v[e] = __float_as_uint(acc[q][h][j0 + j][e] + __uint_as_float(b));
                    }
                    if (tok < a.n && c0 < a.rows) *reinterpret_cast<u32x4m*>(out + ((size_t)tok * a.rows + c0) * SIZE) = v;
                }
        }
    }
}

template <class G>
__global__ __launch_bounds__(G::THREADS, G::PER_SIMD) void mx_tile_kernel(const MxMatArgs a, int n_m, int n_n) {
    extern __shared__ __align__(16) uint8_t s_mem[];
    constexpr int AF = G::AF, Q = G::Q, TN = G::TN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    // an XCD's run of tiles: BAND along the weights by as many as there are along the
    // activations, about as many bytes of one as of the other
    int mt, nt;
    {
        const int lin = xcd_order(blockIdx.x, n_m * n_n), band = lin / (G::BAND * n_n), in = lin - band * G::BAND * n_n, wide = min(G::BAND, n_m - G::BAND * band);
        nt = __builtin_amdgcn_readfirstlane(in / wide);  // (divided on the vector unit)
        mt = __builtin_amdgcn_readfirstlane(G::BAND * band + in - nt * wide);
    }
    const int nblk = a.cols / 32, stages = (nblk + 4 * G::SB - 1) / (4 * G::SB), chunks = (nblk + 15) / 16;
    const int pitch = (int)mx_pitch(a.cols), w_row = a.cols / 2, a_row = (int)mx_row_bytes(AF, a.cols);
    const int col0 = mt * G::COLS, tok0 = nt * G::BN;

    const int cols_in = min(G::COLS, a.rows - col0), toks_in = min(G::BN, a.n - tok0);
    // first output column (within the tile) of weight group q
    auto group_col = [](int q) { return G::GATED ? (q >> 1) * 64 : q * 64; };
    // 16-byte pieces of a stage (buffers over the tile's rows; an instruction's is the wave's own choice)
    __amdgpu_buffer_rsrc_t rw[G::NI_W], rs[G::NI_S];
    const __amdgpu_buffer_rsrc_t ra = tile_rsrc(a.act.codes + (size_t)tok0 * a_row, (size_t)toks_in * a_row);
    constexpr int W_LANES = G::W_ROW / 16, A_LANES = G::A_ROW / 16;  // lanes of a row
    int vw[G::NI_W], bw[G::NI_W], va[G::NI_A], ba[G::NI_A];
#pragma unroll
    for (int k = 0; k < G::NI_W; ++k) {  // LDS row L: row L % 16 of tile L / 16 % 4 of group L / 64
        const int j = wave * G::NI_W + k, L = j * (64 / W_LANES) + lane / W_LANES, R = L & 15;
        const int c = (lane % W_LANES) ^ turn<G::W_ROW>(R);
        vw[k] = (group_col(L >> 6) + 16 * (R >> 2) + 4 * (L >> 4 & 3) + (R & 3)) * w_row + c * 16;
        bw[k] = c;
        const bool second = G::GATED && (j * (64 / W_LANES) >> 6 & 1);  // (a group is whole instructions)
        rw[k] = tile_rsrc((second ? a.up.codes : a.w.codes) + (size_t)col0 * w_row, (size_t)cols_in * w_row);
    }
#pragma unroll
    for (int k = 0; k < G::NI_A; ++k) {
        const int R = (wave * G::NI_A + k) * (64 / A_LANES) + lane / A_LANES, c = (lane % A_LANES) ^ turn<G::A_ROW>(R);
        va[k] = R * a_row + c * 16;
        ba[k] = AF == MX_E4M3 ? c >> 1 : c;
    }
    // scales: 64 rows an instruction, the weight groups' and then the activations'
    int row_s[G::NI_S];
#pragma unroll
    for (int k = 0; k < G::NI_S; ++k) {
        const int j = wave * G::NI_S + k, R = lane & 15, i = lane >> 4;
        row_s[k] = j < G::NSW ? group_col(j) + 16 * (R >> 2) + 4 * i + (R & 3) : (j - G::NSW) * 64 + lane;
        if (j >= G::NSW && row_s[k] >= G::BN) row_s[k] = -1;  // (every wave issues the same number)
        const uint8_t* const base = j >= G::NSW ? a.act.scales : G::GATED && (j & 1) ? a.up.scales : a.w.scales;
        rs[k] = tile_rsrc(base + (size_t)(j >= G::NSW ? tok0 : col0) * pitch, (size_t)(j >= G::NSW ? toks_in : cols_in) * pitch);
    }

    // instruction k of this wave's of stage t, to LDS address `at`
    auto request = [&](int k, int t, uint32_t at) __attribute__((always_inline)) {
        const int left = nblk - 4 * G::SB * t;  // blocks from here on (none: every lane out of range)
        if (k < G::NI_W)
            dma16(rw[k], at + (wave * G::NI_W + k) * 1024, bw[k] < left ? vw[k] : OUT_OF_RANGE, t * G::W_ROW);
        else
            dma16(ra, at + G::W_BYTES + (wave * G::NI_A + k - G::NI_W) * 1024, ba[k - G::NI_W] < left ? va[k - G::NI_W] : OUT_OF_RANGE,
                  t * G::A_ROW);
    };
    auto request_scales = [&](int c, uint32_t at) __attribute__((always_inline)) {  // of chunk c
#pragma unroll
        for (int k = 0; k < G::NI_S; ++k) {
            const MxScalePiece p = mx_scale_piece(row_s[k], pitch, c);
            dma16(rs[k], at + (wave * G::NI_S + k) * 1024, row_s[k] >= 0 && 16 * c < nblk ? p.lane : OUT_OF_RANGE, p.scalar);
        }
    };
    const int wm = wave % G::WM, wn = wave / G::WM;
    f32x4m acc[Q][4][TN] = {};
    // byte offsets of this wave's operands within a stage, and of its scales within a chunk's
    const int at_w = (wm * Q * 64 + r) * G::W_ROW, at_a = G::W_BYTES + (wn * TN * 16 + r) * G::A_ROW;
    const int at_sw = wm * Q * 1024 + r * 16, at_sa = G::NSW * 1024 + wn * TN * 256 + r * 16;
    const int turn_w = turn<G::W_ROW>(r), turn_a = turn<G::A_ROW>(r);

    // operands of the 128 columns s of a stage: tile n % 4 of group n / 4, activation tile j
    auto weights = [&](const uint8_t* st, int s, int n) __attribute__((always_inline)) {
        const u32x4m w = *reinterpret_cast<const u32x4m*>(st + at_w + n * 16 * G::W_ROW + ((4 * s + g) ^ turn_w) * 16);
        return i32x8m{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    };
    auto acts = [&](const uint8_t* st, int s, int j) __attribute__((always_inline)) {
        const uint8_t* const row = st + at_a + j * 16 * G::A_ROW;
        if constexpr (AF == MX_E4M3) {
            const u32x4m lo = *reinterpret_cast<const u32x4m*>(row + ((8 * s + g) ^ turn_a) * 16);
            const u32x4m hi = *reinterpret_cast<const u32x4m*>(row + ((8 * s + 4 + g) ^ turn_a) * 16);
            return i32x8m{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
        } else {
            const u32x4m lo = *reinterpret_cast<const u32x4m*>(row + ((4 * s + g) ^ turn_a) * 16);
            return i32x8m{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], 0, 0, 0, 0};
        }
    };
    // A row's 16 scale bytes -> block g's of each 128 columns.  Behind a row's last block
    // the codes are 0 and so is this (the bytes there are no scales).
    int sw[4 * Q], sa[TN];
    auto scales = [&](int c, const uint8_t* sc) __attribute__((always_inline)) {
        const int left = nblk - 16 * c - g;
        const uint32_t s01 = (left > 0 ? g : 0x0c) | (left > 4 ? 4 + g : 0x0c) << 8 | 0x0c0c0000u;
        const uint32_t s23 = (left > 8 ? g : 0x0c) << 16 | (left > 12 ? 4 + g : 0x0cu) << 24 | 0x0c0cu;
        auto four = [&](int at) __attribute__((always_inline)) {
            const u32x4m d = *reinterpret_cast<const u32x4m*>(sc + at);
            return (int)(__builtin_amdgcn_perm(d[1], d[0], s01) | __builtin_amdgcn_perm(d[3], d[2], s23));
        };
#pragma unroll
        for (int n = 0; n < 4 * Q; ++n) sw[n] = four(at_sw + n * 256);
#pragma unroll
        for (int j = 0; j < TN; ++j) sa[j] = four(at_sa + j * 256);
    };
    auto mfma = [&](auto byte, const i32x8m& w, const i32x8m& o, int n, int j) __attribute__((always_inline)) {
        constexpr int BYTE = decltype(byte)::value;
        f32x4m& d = acc[n / 4][n % 4][j];
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, o, d, 4, AF == MX_E4M3 ? 0 : 4, BYTE, sw[n], BYTE, sa[j]);
    };
    // an activation operand as the MFMA takes it
    constexpr int P = G::SPLIT ? 2 : 1;
    auto parts = [&](const i32x8m& c, i32x8m (&o)[P]) __attribute__((always_inline)) {
        if constexpr (G::SPLIT)
            mx_split(c, o[0], o[1]);
        else
            o[0] = c;
    };
    // The products of a stage, the first of whose 128 columns are number PART of the
    // chunk's; between them `more` (of 4 Q a step) of the DMA of a later one.
    auto multiply = [&](auto part, const uint8_t* st, auto&& more) __attribute__((always_inline)) {
        constexpr int PART = decltype(part)::value;
        if constexpr (G::WHOLE) {
            // few products a step: the next step's operands are on their way before this one's
            i32x8m w[2][4 * Q], o[2][TN];
            auto load = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < TN; ++j) o[s & 1][j] = acts(st, s, j);
#pragma unroll
                for (int n = 0; n < 4 * Q; ++n) w[s & 1][n] = weights(st, s, n);
            };
            load(0);
            static_for<G::SB>([&](auto step) __attribute__((always_inline)) {
                constexpr int S = decltype(step)::value;
                if constexpr (S + 1 < G::SB) load(S + 1);
#pragma unroll
                for (int n = 0; n < 4 * Q; ++n) more(S * 4 * Q + n);
                i32x8m op[TN][P];
#pragma unroll
                for (int j = 0; j < TN; ++j) parts(o[S & 1][j], op[j]);
#pragma unroll
                for (int n = 0; n < 4 * Q; ++n)
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int j = 0; j < TN; ++j) mfma(Int<PART + S>{}, w[S & 1][n], op[j][p], n, j);
                __builtin_amdgcn_sched_barrier(0);
            });
        } else {
            static_for<G::SB>([&](auto step) __attribute__((always_inline)) {
                constexpr int S = decltype(step)::value;
                i32x8m o[TN][P], w = weights(st, S, 0);
#pragma unroll
                for (int j = 0; j < TN; ++j) parts(acts(st, S, j), o[j]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < 4 * Q; ++n) {
                    i32x8m next = w;
                    if (n + 1 < 4 * Q) next = weights(st, S, n + 1);
                    more(S * 4 * Q + n);
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int j = 0; j < TN; ++j) mfma(Int<PART + S>{}, w, o[j][p], n, j);
                    w = next;
                    __builtin_amdgcn_sched_barrier(0);  // or all the DMA would come before all the products
                }
            });
        }
    };

    const uint32_t lds0 = lds_address(s_mem);
#pragma unroll
    for (int c = 0; c < G::AHEAD; ++c) request_scales(c, lds0 + G::S_OFF + c * G::S_STAGE);
#pragma unroll
    for (int s = 0; s < G::STAGES - 1; ++s)
#pragma unroll
        for (int k = 0; k < G::NI; ++k) request(k, s, lds0 + s * G::STAGE);
    int cur = 0, slot = 0, t = 0;
    for (int c = 0; c < chunks; ++c) {
        static_for<G::PARTS>([&](auto of_chunk) __attribute__((always_inline)) {
            constexpr int U = decltype(of_chunk)::value;
            if (U > 0 && t >= stages) return;
            // This wave's pieces of stage t are there, and the chunk's scales, which were asked
            // for before them; behind the barrier everybody's, and everybody has read stage
            // t - 1 and the last chunk's scales, whose places are free.
            wait_vm<(G::STAGES - 2) * G::NI>();
            barrier_lds();
            if constexpr (U == 0) {
                const int behind = slot == 0 ? G::AHEAD : slot - 1;
                scales(c, s_mem + G::S_OFF + slot * G::S_STAGE);
                request_scales(c + G::AHEAD, lds0 + G::S_OFF + behind * G::S_STAGE);
                slot = slot == G::AHEAD ? 0 : slot + 1;
            }
            const int next = cur == 0 ? G::STAGES - 1 : cur - 1;
            constexpr int GAPS = G::SB * 4 * Q, PER = (G::NI + GAPS - 1) / GAPS;  // DMA instructions between two rows of products
            multiply(Int<U * G::SB>{}, s_mem + cur * G::STAGE, [&](int n) __attribute__((always_inline)) {
#pragma unroll
                for (int k = n * PER; k < (n + 1) * PER && k < G::NI; ++k) request(k, t + G::STAGES - 1, lds0 + next * G::STAGE);
            });
            cur = cur == G::STAGES - 1 ? 0 : cur + 1;
            ++t;
        });
    }
    wait_vm<0>();

    // lane (r, g): activation row r of each tile, 16 columns of each group
    const int tok1 = tok0 + wn * TN * 16 + r;
    if constexpr (!G::GATED) {
        const int c1 = col0 + wm * Q * 64 + 16 * g;
        if ((a.rows & 7) == 0 && a.vec) {
            if (a.bf16)
                put_tile<true, Q, TN>(a, acc, tok1, c1);
            else
                put_tile<false, Q, TN>(a, acc, tok1, c1);
            return;
        }
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int tok = tok1 + j * 16, c0 = c1 + q * 64;
                if (tok >= a.n) continue;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + e < a.rows) put_sum(a, (size_t)tok * a.rows + c0 + e, acc[q][e / 4][j][e % 4]);
            }
    } else {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int tok = tok1 + j * 16;
#pragma unroll
            for (int q = 0; q < Q; q += 2) {
                const int c0 = col0 + (wm * Q + q) / 2 * 64 + 16 * g;
                float x[2][8];
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = mx_act(acc[q][e / 4][j][e % 4], a.fn) * acc[q + 1][e / 4][j][e % 4];
                    x[e / 8][e % 8] = v;
                    m = max(m, __float_as_uint(v) & 0x7fffffffu);
                }
                m = max(m, (uint32_t)__shfl_xor((int)m, 16));  // a block: 16 columns of two lane groups
                if (tok >= a.n || c0 >= a.rows) continue;
                uint8_t* const to = a.hidden.codes + (size_t)tok * mx_row_bytes(a.hidden.format, a.rows);
                int byte;
                if (a.hidden.format == MX_E2M1) {
                    byte = mx_scale_byte<MX_E2M1>(m);
                    *reinterpret_cast<u32x2m*>(to + c0 / 2) = u32x2m{mx_encode8<MX_E2M1>(x[0], byte)[0], mx_encode8<MX_E2M1>(x[1], byte)[0]};
                } else {
                    byte = mx_scale_byte<MX_E4M3>(m);
                    const u32x2m lo = mx_encode8<MX_E4M3>(x[0], byte), hi = mx_encode8<MX_E4M3>(x[1], byte);
                    *reinterpret_cast<u32x4m*>(to + c0) = u32x4m{lo[0], lo[1], hi[0], hi[1]};
                }
                if ((g & 1) == 0) a.hidden.scales[(size_t)tok * mx_pitch(a.rows) + c0 / 32] = (uint8_t)byte;
            }
        }
    }
}

template <class G>
hipError_t tile(const MxMatArgs& a, hipStream_t st) {
    const int n_m = (a.rows + G::COLS - 1) / G::COLS, n_n = (a.n + G::BN - 1) / G::BN;
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(mx_tile_kernel<G>), hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((mx_tile_kernel<G>), dim3((unsigned)(n_m * n_n)), dim3(G::THREADS), G::LDS, st, a, n_m, n_n);
    return hipGetLastError();
}

//                              AF, gated, WM, Q, WN, TN, SB, STAGES
template <int AF, bool GATED>
hipError_t tiles(int kernel, const MxMatArgs& a, hipStream_t st) {
    constexpr bool EIGHT = AF == MX_E4M3;
    // Where no CU gets a second tile, a tile takes the LDS of two.  Weights that no cache holds,
    // gated, 8 bit codes, 64 x 64 tiles: 64 rows through 12288 x 4096 20.6 us (two stages 25.7; 128 rows,
    // two tiles a CU, 36.9 and 30.3), 64 x 128: 128 rows 32.9 (32.4; 512 rows 94 and 80; in one part, as 4
    // bit codes, 22.6 and 26.4, 58 and 54).  Products, 64 x 64: 256 rows through 4096 x 12288 27.0 (four stages of half as many columns 29.5).
    auto one = [&](int columns, int acts) { return ((a.rows + columns - 1) / columns) * (long)((a.n + acts - 1) / acts) <= a.n_cu; };
    switch (kernel) {
        case MX_KERNEL_64x64:
            if constexpr (GATED)
                return one(64, 64) ? tile<TileGeom<AF, true, 1, 2, 4, 1, 2, 3>>(a, st) : tile<TileGeom<AF, true, 1, 2, 4, 1, 2, 2>>(a, st);
            else
                return tile<TileGeom<AF, false, 1, 1, 4, 1, 4, 3>>(a, st);
        case MX_KERNEL_64x128:
            if constexpr (GATED)
                return one(64, 128) ? tile<TileGeom<AF, true, 1, 2, 4, 2, 2, 3>>(a, st) : tile<TileGeom<AF, true, 1, 2, 4, 2, 1, 3>>(a, st);
            else
                return tile<TileGeom<AF, false, 1, 1, 4, 2, 2, 3>>(a, st);
        // Stages that fill LDS: 4 bit codes, gated, 1024 rows through 12288 x 4096 72 us (two stages 79).
        case MX_KERNEL_256x128: return tile<TileGeom<AF, GATED, 2, 2, 4, 2, 2, EIGHT ? 2 : 3>>(a, st);
        // 8 bit codes: three stages of 128 columns fill LDS.  4 bit: two of 256 (2553 rows
        // through 18944 x 3584 124 us, three of 128 130 us).
        case MX_KERNEL_256x256: return tile<TileGeom<AF, GATED, 2, 2, 4, 4, EIGHT ? 1 : 2, EIGHT ? 3 : 2>>(a, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_mx_tile(int kernel, const MxMatArgs& a, hipStream_t st) {
    if (a.act.format == MX_E4M3) return a.gated ? tiles<MX_E4M3, true>(kernel, a, st) : tiles<MX_E4M3, false>(kernel, a, st);
    return a.gated ? tiles<MX_E2M1, true>(kernel, a, st) : tiles<MX_E2M1, false>(kernel, a, st);
}

}  // namespace dr
