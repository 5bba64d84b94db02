// mx_ring.hip -- products of E2M1 weights with microscaled activations, few rows:
// a workgroup's waves share a strip of weight rows and up to 64 activation rows
// and split the columns; each wave streams its own part through LDS, and the
// sums are joined there at the end, in a fixed order.
//
// With few rows the weights' bytes bound the product, or the latency of the few
// steps a workgroup takes: what counts is how many bytes are under way, in as many
// workgroups as a CU holds (direct loads into registers, with half as many waves: 21.5
// us for one row through 2 x 12288 x 4096 against 12.1, 79 us for 256 rows through 4096 x
// 4096 against 13.3; the large copy's rate allows 11.2 and 3.9).  Each wave
// keeps STAGES steps of weights, activations and scales in flight by LDS DMA
// (whole rows of 64 or 128 bytes, consecutive lanes on consecutive bytes), waits for
// nobody but its own loads and meets the others once, at the end.
//
// EXACT: both operands are turned into bf16, which holds every code times its
// power of two exactly (blocks of scale bytes 3 to 246; below, 8 bit codes' values can lie
// under its smallest number, and above, the largest codes become infinite), and multiplied by the bf16 MFMA, whose sums keep f32's
// bits, where the block-scaled MFMA drops some of 8 bit codes' (mx_split: over 4096 columns
// relative errors of 4e-6 to 5e-5 against 1e-7).  Taken for f32 outputs of 8 bit codes, and wherever
// the conversions hide behind the loads.  A product does not depend on the order of the columns, so
// the MFMA's k index is whatever both operands agree on: lane group g takes block g
// of a step's four, and instruction j multiplies the blocks' values 8 j .. 8 j + 7.
#include <climits>

#include "mx_common.hpp"

namespace dr {
namespace {

__device__ __forceinline__ bf16x8m join(bf16x2 a, bf16x2 b, bf16x2 c, bf16x2 d) {
    return bf16x8m{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// A block's 32 values as four operands.
__device__ __forceinline__ void operands4(const u32x4m& c, float s, bf16x8m (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        o[j] = join(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], s, 1),
                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], s, 3));
}
__device__ __forceinline__ void operands8(const u32x4m (&c)[2], float s, bf16x8m (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = c[j / 2][2 * (j & 1)], b = c[j / 2][2 * (j & 1) + 1];
        o[j] = join(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true),
                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true));
    }
}

// MT tiles of 16 weight rows (gated: the first half of the gate, the second of the up
// projection, of the same output columns) by NT tiles of 16 activation rows, of which
// AR are staged (a multiple of 4; fewer than 16 with one tile); steps of SK * 128 columns.
template <int AF_, bool GATED_, bool EXACT_, int MT_, int NT_, int AR_, int SK_, int STAGES_, int WAVES_>
struct RingGeom {
    static constexpr int AF = AF_, MT = MT_, NT = NT_, AR = AR_, SK = SK_, STAGES = STAGES_, WAVES = WAVES_;
    static constexpr bool GATED = GATED_, EXACT = EXACT_;
    static constexpr int FT = GATED ? MT / 2 : MT;  // tiles of output columns
    static constexpr bool PAIRS = EXACT && AF == MX_E4M3;
    static constexpr int W_ROW = SK * 64, A_ROW = SK * (AF == MX_E4M3 ? 128 : 64);  // bytes of a row and step
    static constexpr int NW = MT * 16 * W_ROW / 1024;                               // DMA instructions of a step
    static constexpr int NA = (AR * A_ROW + 1023) / 1024;
    static constexpr int NSM = (FT * 16 * SK + 63) / 64;  // scales of one matrix
    static constexpr int NSW = GATED ? 2 * NSM : NSM, NSA = (AR * SK + 63) / 64;
    static constexpr int NI = NW + NA + NSW + NSA;
    static constexpr int A_OFF = NW * 1024, SW_OFF = A_OFF + NA * 1024, SA_OFF = SW_OFF + NSW * 256, STAGE = SA_OFF + NSA * 256;
    static constexpr int TILE = 16 * 20;  // floats of a tile of sums: rows of 16 and 4 apart
    static constexpr int RING = STAGE * STAGES * WAVES, SUMS = WAVES * MT * NT * TILE * 4;
    static constexpr int LDS = RING > SUMS ? RING : SUMS;
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert(!GATED || FT % 2 == 0, "whole blocks of output columns");
    static_assert((STAGES - 1) * NI < 64, "vmcnt");
    static_assert(NT * 16 == AR || (NT == 1 && (AR == 4 || AR == 8)), "staged rows");
};

template <class G>
__global__ __launch_bounds__(64 * G::WAVES) void mx_ring_kernel(const MxMatArgs a, int groups) {
    extern __shared__ __align__(16) uint8_t s_mem[];
    constexpr int AF = G::AF, MT = G::MT, NT = G::NT, SK = G::SK, WAVES = G::WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    // (an XCD takes a strip's groups of activation rows one after the other)
    const int lin = xcd_order(blockIdx.x, gridDim.x), strip = __builtin_amdgcn_readfirstlane(lin / groups);
    const int col0 = strip * G::FT * 16, tok0 = __builtin_amdgcn_readfirstlane(lin - strip * groups) * NT * 16;
    const int nblk = a.cols / 32, steps = (nblk + 4 * SK - 1) / (4 * SK);
    const int pitch = (int)mx_pitch(a.cols), w_row = a.cols / 2, a_row = (int)mx_row_bytes(AF, a.cols);
    const int cols_in = min(G::FT * 16, a.rows - col0), toks_in = min(G::NT * 16, a.n - tok0);

    const __amdgpu_buffer_rsrc_t rw = tile_rsrc(a.w.codes + (size_t)col0 * w_row, (size_t)cols_in * w_row);
    const __amdgpu_buffer_rsrc_t rws = tile_rsrc(a.w.scales + (size_t)col0 * pitch, (size_t)cols_in * pitch);
    const __amdgpu_buffer_rsrc_t ru = tile_rsrc((G::GATED ? a.up : a.w).codes + (size_t)col0 * w_row, (size_t)cols_in * w_row);
    const __amdgpu_buffer_rsrc_t rus = tile_rsrc((G::GATED ? a.up : a.w).scales + (size_t)col0 * pitch, (size_t)cols_in * pitch);
    const __amdgpu_buffer_rsrc_t ra = tile_rsrc(a.act.codes + (size_t)tok0 * a_row, (size_t)toks_in * a_row);
    const __amdgpu_buffer_rsrc_t ras = tile_rsrc(a.act.scales + (size_t)tok0 * pitch, (size_t)toks_in * pitch);

    // Lane addresses of a step's pieces (row in the strip, piece in the row).
    constexpr int W_LANES = G::W_ROW / 16, A_LANES = G::A_ROW / 16;  // lanes of a row
    constexpr int W_ROWS = 64 / W_LANES, A_ROWS = 64 / A_LANES;      // rows of an instruction
    constexpr int NWM = G::FT * 16 / W_ROWS;                         // instructions of one matrix
    int vw[NWM], bw[NWM], va[G::NA], ba[G::NA], vsw[G::NSM], vsa[G::NSA];
#pragma unroll
    for (int k = 0; k < NWM; ++k) {
        const int R = k * W_ROWS % 16 + lane / W_LANES, c = (lane % W_LANES) ^ turn<G::W_ROW>(R);
        vw[k] = (R + k * W_ROWS / 16 * 16) * w_row + c * 16;
        bw[k] = c;
    }
#pragma unroll
    for (int k = 0; k < G::NA; ++k) {
        const int R = k * A_ROWS % 16 + lane / A_LANES, c = (lane % A_LANES) ^ turn<G::A_ROW, G::PAIRS>(R);
        va[k] = R + k * A_ROWS / 16 * 16 < G::AR ? (R + k * A_ROWS / 16 * 16) * a_row + c * 16 : OUT_OF_RANGE;
        ba[k] = AF == MX_E4M3 ? c >> 1 : c;
    }
    // scale bytes: dword SK * R + s is row R's of the step's 128 columns s
    const int ss = lane % SK;
#pragma unroll
    for (int k = 0; k < G::NSM; ++k) {
        const int R = (k * 64 + lane) / SK;
        vsw[k] = R < G::FT * 16 ? R * pitch + ss * 4 : OUT_OF_RANGE;
    }
#pragma unroll
    for (int k = 0; k < G::NSA; ++k) {
        const int R = (k * 64 + lane) / SK;
        vsa[k] = R < G::AR ? R * pitch + ss * 4 : OUT_OF_RANGE;
    }
    const uint32_t ring = lds_address(s_mem) + wave * G::STAGES * G::STAGE;
    auto request = [&](int t, uint32_t at) __attribute__((always_inline)) {
        const int left = nblk - 4 * SK * t;  // blocks from here on (none: every lane out of range)
#pragma unroll
        for (int k = 0; k < G::NW; ++k)
            dma16(k >= NWM ? ru : rw, at + k * 1024, bw[k % NWM] < left ? vw[k % NWM] : OUT_OF_RANGE, t * G::W_ROW);
#pragma unroll
        for (int k = 0; k < G::NA; ++k) dma16(ra, at + G::A_OFF + k * 1024, ba[k] < left ? va[k] : OUT_OF_RANGE, t * G::A_ROW);
#pragma unroll
        for (int k = 0; k < G::NSW; ++k)
            dma4(k >= G::NSM ? rus : rws, at + G::SW_OFF + k * 256, 4 * ss < left ? vsw[k % G::NSM] : OUT_OF_RANGE, t * SK * 4);
#pragma unroll
        for (int k = 0; k < G::NSA; ++k)
            dma4(ras, at + G::SA_OFF + k * 256, 4 * ss < left ? vsa[k] : OUT_OF_RANGE, t * SK * 4);
    };

    // A step's operands, from LDS: weight tile i (block g of each 128 columns s), activation
    // tile j, and the scale bytes of block g.
    u32x4m cw[SK][MT], ca[SK][NT][AF == MX_E4M3 ? 2 : 1];
    int sw[SK][MT], sa[SK][NT];
    auto load = [&](int t, const uint8_t* st) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < SK; ++s) {
            // behind a row's last block the codes are 0 and so is its byte (the bytes there are no scales)
            const uint32_t sel = 4 * (SK * t + s) + g < nblk ? 0x0c0c0c00u | g : 0x0c0c0c0cu;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int R = G::AR < 16 ? r & (G::AR - 1) : r;  // (the other rows' sums are not used)
                const uint8_t* const row = st + G::A_OFF + (j * 16 + R) * G::A_ROW;
                const int x = turn<G::A_ROW, G::PAIRS>(R);
                if constexpr (AF == MX_E4M3) {
                    const int c = 8 * s + (G::EXACT ? 2 * g : g);
                    ca[s][j][0] = *reinterpret_cast<const u32x4m*>(row + (c ^ x) * 16);
                    ca[s][j][1] = *reinterpret_cast<const u32x4m*>(row + ((c + (G::EXACT ? 1 : 4)) ^ x) * 16);
                } else {
                    ca[s][j][0] = *reinterpret_cast<const u32x4m*>(row + ((4 * s + g) ^ x) * 16);
                }
                sa[s][j] = (int)__builtin_amdgcn_perm(0, *reinterpret_cast<const uint32_t*>(st + G::SA_OFF + ((j * 16 + R) * SK + s) * 4), sel);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                cw[s][i] = *reinterpret_cast<const u32x4m*>(st + (i * 16 + r) * G::W_ROW + ((4 * s + g) ^ turn<G::W_ROW>(r)) * 16);
                sw[s][i] = (int)__builtin_amdgcn_perm(
                    0, *reinterpret_cast<const uint32_t*>(st + G::SW_OFF + i / G::FT * G::NSM * 256 + ((i % G::FT * 16 + r) * SK + s) * 4), sel);
            }
        }
    };
    f32x4m acc[MT][NT] = {};
    auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < SK; ++s) {
            bf16x8m oa[NT][4];
            if constexpr (G::EXACT) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (AF == MX_E4M3)
                        operands8(ca[s][j], mx_scale(sa[s][j]), oa[j]);
                    else
                        operands4(ca[s][j][0], mx_scale(sa[s][j]), oa[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const u32x4m& w = cw[s][i];
                if constexpr (G::EXACT) {
                    bf16x8m ow[4];
                    operands4(w, mx_scale(sw[s][i]), ow);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ow[q], oa[j][q], acc[i][j], 0, 0, 0);
                } else {
                    const i32x8m ow = i32x8m{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const u32x4m &lo = ca[s][j][0], &hi = ca[s][j][AF == MX_E4M3 ? 1 : 0];
                        const i32x8m o = AF == MX_E4M3 ? i32x8m{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]}
                                                       : i32x8m{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], 0, 0, 0, 0};
                        auto add = [&](const i32x8m& x) __attribute__((always_inline)) {
                            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ow, x, acc[i][j], 4, AF == MX_E4M3 ? 0 : 4, 0, sw[s][i], 0, sa[s][j]);
                        };
                        if constexpr (G::GATED && AF == MX_E4M3) {
                            i32x8m large, small;
                            mx_split(o, large, small);  // (once for all weight tiles)
                            add(large);
                            add(small);
                        } else {
                            add(o);
                        }
                    }
                }
            }
        }
    };

    // Wave w takes steps w, w + WAVES, ...  A step's operands wait in registers while it is
    // multiplied, so that its place in the ring is on its way again meanwhile.
#pragma unroll
    for (int s = 0; s < G::STAGES; ++s) request(wave + s * WAVES, ring + s * G::STAGE);
    int cur = 0;
    for (int t = wave; t < steps; t += WAVES) {
        wait_vm<(G::STAGES - 1) * G::NI>();
        load(t, s_mem + (wave * G::STAGES + cur) * G::STAGE);
        wait_lds();
        request(t + G::STAGES * WAVES, ring + cur * G::STAGE);
        multiply();
        cur = cur == G::STAGES - 1 ? 0 : cur + 1;
    }
    wait_vm<0>();
    barrier_lds();  // no wave reads or fills the rings any more

    // lane (r, g) holds weight rows 4 g .. 4 g + 3 of each tile for activation row r
    float* const s_sum = reinterpret_cast<float*>(s_mem);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<f32x4m*>(s_sum + ((wave * MT + i) * NT + j) * G::TILE + r * 20 + 4 * g) = acc[i][j];
    barrier_lds();
    auto total = [&](int tile, int quad, int t) __attribute__((always_inline)) {
        f32x4m x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            x = x + *reinterpret_cast<const f32x4m*>(s_sum + ((w * MT + tile) * NT + t / 16) * G::TILE + t % 16 * 20 + 4 * quad);
        return x;
    };
    constexpr int QUADS = G::FT * 4;
    for (int e = threadIdx.x; e < QUADS * NT * 16; e += 64 * WAVES) {  // (whole waves)
        const int f = e % QUADS, t = e / QUADS, c0 = col0 + 4 * f, tok = tok0 + t;
        const f32x4m x = total(f / 4, f % 4, t);
        const bool in = tok < a.n && c0 < a.rows;
        if constexpr (!G::GATED) {
            if (!in) continue;
            const size_t at = (size_t)tok * a.rows + c0;
            if (a.vec && (a.rows & 3) == 0) {
                f32x4m y = x;
                if (a.bf16) {
                    if (a.residual) {
                        const u32x2m v = *reinterpret_cast<const u32x2m*>(static_cast<const uint16_t*>(a.residual) + at);
                        y = y + f32x4m{mx_f32(v[0] & 0xffff), __uint_as_float(v[0] & 0xffff0000u), mx_f32(v[1] & 0xffff),
                                       __uint_as_float(v[1] & 0xffff0000u)};
                    }
                    *reinterpret_cast<u32x2m*>(static_cast<uint16_t*>(a.out) + at) =
                        u32x2m{mx_bf16(y[0]) | (uint32_t)mx_bf16(y[1]) << 16, mx_bf16(y[2]) | (uint32_t)mx_bf16(y[3]) << 16};
                } else {
                    if (a.residual) y = y + *reinterpret_cast<const f32x4m*>(static_cast<const float*>(a.residual) + at);
                    *reinterpret_cast<f32x4m*>(static_cast<float*>(a.out) + at) = y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c0 + i < a.rows) put_sum(a, at + i, x[i]);
            }
        } else {
            const f32x4m u = total(G::FT + f / 4, f % 4, t);
            float v[4];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = mx_act(x[i], a.fn) * u[i];
                m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            m = quad_max(m);
            m = max(m, (uint32_t)__shfl_xor((int)m, 4));  // a block: 8 lanes' 32 columns
            if (!in) continue;
            uint8_t* const to = a.hidden.codes + (size_t)tok * mx_row_bytes(a.hidden.format, a.rows);
            int byte;
            if (a.hidden.format == MX_E2M1) {
                byte = mx_scale_byte<MX_E2M1>(m);
                *reinterpret_cast<uint16_t*>(to + c0 / 2) = (uint16_t)mx_encode4<MX_E2M1>(v, byte);
            } else {
                byte = mx_scale_byte<MX_E4M3>(m);
                *reinterpret_cast<uint32_t*>(to + c0) = mx_encode4<MX_E4M3>(v, byte);
            }
            if ((f & 7) == 0) a.hidden.scales[(size_t)tok * mx_pitch(a.rows) + c0 / 32] = (uint8_t)byte;
        }
    }
}

template <class G>
hipError_t ring(const MxMatArgs& a, hipStream_t st) {
    const int groups = (a.n + G::NT * 16 - 1) / (G::NT * 16), strips = (a.rows + G::FT * 16 - 1) / (G::FT * 16);
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(mx_ring_kernel<G>), hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((mx_ring_kernel<G>), dim3((unsigned)groups * strips), dim3(64 * G::WAVES), G::LDS, st, a, groups);
    return hipGetLastError();
}

//                              AF, gated, exact, MT, NT, AR, SK, STAGES, WAVES
template <int AF, bool X>
hipError_t launch(int kernel, const MxMatArgs& a, hipStream_t st) {
    // One place in the ring (and a step in registers): one row through 2 x 12288 x 4096 12.1 us
    // (4.4 TB/s of weights, which the memory-side cache holds; 14.6 from memory), 4096 x 12288
    // 7.2, 16 rows 12.7 and 8.2; two places 13.2, 7.3, 15.9 and 8.7: fewer workgroups fit on a
    // CU.  Where no CU gets a second workgroup and there
    // are steps for all, twice the waves keep as many bytes under way as two would.  With weights
    // that no cache holds: one row through 3584 x 18944 9.5 us (8 waves 11.9; 10.3 and 11.0 on another
    // day), 4096 x 12288 7.8 (8.7), 2048 x 8192 5.5 (6.3); held by the memory-side cache 8.7 (9.0; 8.5 and 8.2),
    // 7.2 (7.1) and 5.0 (4.8): a layer's weights come from memory.  2 x 4096 x 4096, from
    // memory, 7.8 (4 waves 9.4), 2 x 8192 x 4096 9.6 (11.6); with more columns
    // they take away workgroups instead, 2 x 9216 x 4096 16 rows 17.3 (15.7), one row 5120 x 8192
    // 9.1 (8.3), and with fewer steps they have none, 2 x 1024 x 1024 4.2 (4.0).
    if constexpr (X || AF == MX_E2M1) {
        const int steps = (a.cols + 255) / 256;
        const bool one = (a.rows + (a.gated ? 31 : 15)) / (a.gated ? 32 : 16) <= a.n_cu;
        if (kernel == MX_KERNEL_4) {
            if (a.gated && one && steps >= 8) return ring<RingGeom<AF, true, X, 4, 1, 4, 2, 1, 8>>(a, st);
            if (a.gated) return ring<RingGeom<AF, true, X, 4, 1, 4, 2, 1, 4>>(a, st);
            if (one && steps >= 32) return ring<RingGeom<AF, false, X, 1, 1, 4, 2, 1, 16>>(a, st);
            return ring<RingGeom<AF, false, X, 1, 1, 4, 2, 1, 8>>(a, st);
        }
        if (kernel == MX_KERNEL_16) {
            if (a.gated && one && steps >= 8) return ring<RingGeom<AF, true, X, 4, 1, 16, 2, 1, 8>>(a, st);
            if (a.gated) return ring<RingGeom<AF, true, X, 4, 1, 16, 2, 1, 4>>(a, st);
            // 16 rows' bytes and conversions are as much as 32 weight rows': where a CU gets more than
            // 16 columns, it reads them once for 32 (8192 x 8192 11.1 us, 16 a time 13.5; 65536 x 4096
            // 37.9 and 46.4; 4096 x 12288 13.4 and 10.7, half the CUs have none).
            return one ? ring<RingGeom<AF, false, X, 1, 1, 16, 2, 1, 8>>(a, st) : ring<RingGeom<AF, false, X, 2, 1, 16, 2, 1, 8>>(a, st);
        }
    }
    if constexpr (X) {
        if (kernel == MX_KERNEL_64x64_EXACT) return ring<RingGeom<AF, false, X, 4, 4, 64, 1, 1, 8>>(a, st);
    } else {
        if (a.gated && kernel == MX_KERNEL_32x32) return ring<RingGeom<AF, true, X, 4, 2, 32, 1, 2, 4>>(a, st);
    }
    if (kernel == MX_KERNEL_16x32) return ring<RingGeom<AF, false, X, 1, 2, 32, 2, 1, 8>>(a, st);
    if (kernel == MX_KERNEL_32x32) return ring<RingGeom<AF, false, X, 2, 2, 32, 1, 1, 8>>(a, st);
    if (kernel == MX_KERNEL_64x32) return ring<RingGeom<AF, false, X, 4, 2, 32, 1, 1, 8>>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace

// The kernel for a product.  Up to 16 rows: strips of 16 or 32 weight rows (gated: 32 of
// either projection), with 4 or 16 activation rows staged.  More: the kernel whose
// estimate is least.  An estimate is a start and, for each round of workgroups that
// the device holds at once, a time per 128 columns; nanoseconds fitted to 17 to 2048
// rows through 1024 x 2048 to 18944 x 3584, which they meet to about 20 %:
//                         start  per round and 128 columns
//   16 x 32                2500    90   4096 x 4096, 32 rows 5.5 us, 4096 x 12288 10.7
//   32 x 32                2500   110   (gated 200) 64 rows 6.3 and 13.1; 12288 x 4096 gated, 32 rows 15.3
//   64 x 32                2500   170   (bf16 MFMA 185) 128 rows 8.1 and 18.3 (32 x 32: 9.4 and 22.4; 64 x 64: 9.5 and 21)
//   64 x 64, bf16 MFMA     2500   340   f32 outputs of 8 bit codes; 256 rows 13.5 and 30
//   64 x 64                2500   220   256 rows 9.7 and 21.2
//   64 x 128               4500   285   512 rows 13.3 and 31.4 (64 x 64: 17.6 and 40.6)
//   256 x 128              4000   880   (700 where at most 3/4 of the CUs have one) 2048 rows 33 and 81, 1024 rows 26 and 65
//   256 x 256              8000  1350   4096 x 12288, 4096 rows 155
// gated, 4 bit codes (fitted to 8 bit ones in one part), and 8 bit codes, whose products are
// two MFMAs; 12288 x 4096, 8 bit:
//   64 x 64, 2 a CU        2500   500   760 (385, 550 where one is enough) 128 rows 26.8 us, 64 rows 20.1
//   64 x 128, 2 a CU       2500   880  1420 (490, 900 + 910 where one is enough) 512 rows 78, 256 rows 47, 128 rows 31.6
//   256 x 128              4000   880  1400 (128 output columns; 700, 1210 where at most 3/4 of the CUs have one) 256 rows 47
//   256 x 256              8000  1350  2400
// Both sides of a step: 256 rows: 256 x 128 46.7 us, 256 x 256 85, 64 x 128 46.7, 64 x 64 43.5; 1024 rows:
// 256 x 128 149, 256 x 256 171; 2048 rows: 295, 272; 4096 x 2048, 128 rows: 32 x 32 8.4, 64 x 64 11.0.
int mx_plan(bool gated, bool exact, int rows, int cols, int n, int n_cu) {
    if (n <= 16) return n <= 4 ? MX_KERNEL_4 : MX_KERNEL_16;
    const long steps = (cols + 127) / 128;
    int best = 0;
    long least = LONG_MAX;
    auto tiles = [&](int columns, int acts) { return (long)((rows + columns - 1) / columns) * ((n + acts - 1) / acts); };
    auto offer = [&](int kernel, int columns, int acts, int per_cu, long start, long step) {
        const long t = start + (tiles(columns, acts) + (long)per_cu * n_cu - 1) / ((long)per_cu * n_cu) * steps * step;
        if (t < least) least = t, best = kernel;
    };
    if (gated && exact) {
        const bool one = tiles(64, 128) <= n_cu;
        offer(MX_KERNEL_32x32, 32, 32, 1, 2500, 200);
        offer(MX_KERNEL_64x64, 64, 64, 2, 2500, tiles(64, 64) <= n_cu ? 550 : 760);
        offer(MX_KERNEL_64x128, 64, 128, 2, one ? 900 : 2500, one ? 910 : 1420);
        offer(MX_KERNEL_256x128, 128, 128, 1, 4000, 4 * tiles(128, 128) <= 3 * n_cu ? 1210 : 1400);
        offer(MX_KERNEL_256x256, 128, 256, 1, 8000, 2400);
    } else if (gated) {
        offer(MX_KERNEL_32x32, 32, 32, 1, 2500, 200);
        offer(MX_KERNEL_64x64, 64, 64, 2, 2500, tiles(64, 64) <= n_cu ? 385 : 500);
        offer(MX_KERNEL_64x128, 64, 128, 2, 2500, tiles(64, 128) <= n_cu ? 490 : 880);
        offer(MX_KERNEL_256x128, 128, 128, 1, 4000, 4 * tiles(128, 128) <= 3 * n_cu ? 700 : 880);
        offer(MX_KERNEL_256x256, 128, 256, 1, 8000, 1350);
    } else {
        offer(MX_KERNEL_16x32, 16, 32, 1, 2500, 90);
        offer(MX_KERNEL_32x32, 32, 32, 1, 2500, 110);
        offer(MX_KERNEL_64x32, 64, 32, 1, 2500, exact ? 185 : 170);
        if (exact) {
            offer(MX_KERNEL_64x64_EXACT, 64, 64, 1, 2500, 340);
        } else {
            offer(MX_KERNEL_64x64, 64, 64, 1, 2500, 220);
            offer(MX_KERNEL_64x128, 64, 128, 1, 4500, 285);
            offer(MX_KERNEL_256x128, 256, 128, 1, 4000, 4 * tiles(256, 128) <= 3 * n_cu ? 700 : 880);
            offer(MX_KERNEL_256x256, 256, 256, 1, 8000, 1350);
        }
    }
    return best;
}

hipError_t launch_mx_matmul(const MxMatArgs& a, hipStream_t st) {
    if (a.n <= 0 || a.rows <= 0) return hipSuccess;
    const bool eight = a.act.format == MX_E4M3;
    // f32 outputs of 8 bit codes stay on the bf16 MFMA; so do bf16 outputs and the gated block up
    // to 16 rows, where the conversions hide behind the weights.  The gated block of more rows
    // multiplies 8 bit codes in two parts (mx_split).
    const bool exact = eight && !a.gated && !a.bf16;
    const int kernel = mx_plan(a.gated, eight && (a.gated || !a.bf16), a.rows, a.cols, a.n, a.n_cu);
    if (kernel > MX_KERNEL_64x64_EXACT) return launch_mx_tile(kernel, a, st);
    if (!eight) return launch<MX_E2M1, false>(kernel, a, st);
    if (exact || kernel <= MX_KERNEL_16) return launch<MX_E4M3, true>(kernel, a, st);
    return launch<MX_E4M3, false>(kernel, a, st);
}

}  // namespace dr
