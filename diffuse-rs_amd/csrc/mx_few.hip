// mx_few.hip -- products of E2M1 weights with microscaled activations: a
// workgroup's eight waves share a strip of weight rows and 16 activation rows,
// each wave a part of the columns, joined through LDS in a fixed order.
//
// Both operands are turned into bf16, which holds every code times its power of
// two exactly, and multiplied by the bf16 MFMA, whose sums keep f32's bits: the
// 8 bit MFMA lines the products of a step up with the largest and drops what
// lies more than about 2^19 below it (relative errors of 4e-6 to 5e-5 against
// 1e-7, measured over 4096 columns).
//
// A step is 512 columns, 16 blocks: lane (r, g) = (lane % 16, lane / 16) takes
// blocks 4 g .. 4 g + 3 of weight row r and of activation row r: 64 and 128 (or
// 64) consecutive bytes, and one aligned load of four scale bytes.  A product
// does not depend on the order of the columns, so the MFMA's k index is whatever
// both operands agree on: instruction j of block s multiplies values 8 j .. 8 j + 7
// of block 4 g + s in lane group g.
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

// MT tiles of 16 weight rows (gated: the first half of the gate, the second of
// the up projection) by 16 activation rows.
template <int AF, bool GATED, int MT>
__global__ __launch_bounds__(512) void mx_few_kernel(const MxMatArgs a) {
    constexpr int ROW = 20;  // floats between a tile's activation rows in LDS
    constexpr int FT = GATED ? MT / 2 : MT;  // feature tiles of the strip
    __shared__ __align__(16) float s_sum[8][MT][16 * ROW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int strips = (a.rows + FT * 16 - 1) / (FT * 16);
    const int tg = blockIdx.x / strips, strip = (blockIdx.x - tg * strips) * FT * 16, tok0 = tg * 16;
    const int nblk = a.cols / 32, steps = (nblk + 15) / 16;
    const size_t pitch = mx_pitch(a.cols), w_row = a.cols / 2, a_row = mx_row_bytes(AF, a.cols);

    const uint8_t* wp[MT];
    const uint8_t* ws[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const MxRows& w = GATED && i >= FT ? a.up : a.w;
        const size_t row = min(strip + (i % FT) * 16 + r, a.rows - 1);  // (rows behind the last: not written)
        wp[i] = w.codes + row * w_row;
        ws[i] = w.scales + row * pitch;
    }
    const int tok = tok0 + r;
    const bool live = tok < a.n;  // other lanes' operands are 0
    const uint8_t* ap = a.act.codes + (size_t)(live ? tok : 0) * a_row;
    const uint8_t* as = a.act.scales + (size_t)(live ? tok : 0) * pitch;

    f32x4m acc[MT] = {};
    for (int t = wave; t < steps; t += 8) {
        const int b0 = t * 16 + 4 * g;
        uint32_t sw[MT], sa = 0;
        u32x4m cw[MT][4], ca[4][AF == MX_E4M3 ? 2 : 1];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bool in = b0 + s < nblk;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                cw[i][s] = u32x4m{0, 0, 0, 0};
                if (in) cw[i][s] = *reinterpret_cast<const u32x4m*>(wp[i] + (size_t)(b0 + s) * 16);
            }
#pragma unroll
            for (int h = 0; h < (AF == MX_E4M3 ? 2 : 1); ++h) {
                ca[s][h] = u32x4m{0, 0, 0, 0};
                if (in && live) ca[s][h] = *reinterpret_cast<const u32x4m*>(ap + (size_t)(b0 + s) * (AF == MX_E4M3 ? 32 : 16) + h * 16);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sw[i] = 0;
            if (b0 < nblk) sw[i] = *reinterpret_cast<const uint32_t*>(ws[i] + b0);
        }
        if (b0 < nblk && live) sa = *reinterpret_cast<const uint32_t*>(as + b0);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bool in = b0 + s < nblk;  // (scale bytes behind a row's last block are not read as scales)
            bf16x8m oa[4];
            const float fa = in && live ? mx_scale((sa >> (8 * s)) & 255) : 1.0f;
            if constexpr (AF == MX_E4M3)
                operands8(ca[s], fa, oa);
            else
                operands4(ca[s][0], fa, oa);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                bf16x8m ow[4];
                operands4(cw[i][s], in ? mx_scale((sw[i] >> (8 * s)) & 255) : 1.0f, ow);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ow[j], oa[j], acc[i], 0, 0, 0);
            }
        }
    }
    // lane (r, g) holds weight rows 4 g .. 4 g + 3 of each tile for activation row r
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4m*>(&s_sum[wave][i][r * ROW + 4 * g]) = acc[i];
    __syncthreads();
    auto total = [&](int tile, int f, int t) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) x += s_sum[w][tile][t * ROW + f];
        return x;
    };
    if constexpr (!GATED) {
        for (int e = threadIdx.x; e < MT * 256; e += 512) {
            const int f = e % (MT * 16), t = e / (MT * 16);
            if (strip + f >= a.rows || tok0 + t >= a.n) continue;
            put_sum(a, (size_t)(tok0 + t) * a.rows + strip + f, total(f / 16, f % 16, t));
        }
    } else {
        static_assert(!GATED || MT == 4, "a strip is one block of the output");
        const int f = threadIdx.x & 31, t = threadIdx.x >> 5;
        const float x = mx_act(total(f / 16, f % 16, t), a.fn) * total(2 + f / 16, f % 16, t);
        uint32_t m = __float_as_uint(x) & 0x7fffffffu;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __shfl(x, (lane & 32) + ((f & 3) * 8) + i);
        const bool row_in = tok0 + t < a.n;
        const size_t at = (size_t)(tok0 + t) * mx_row_bytes(a.hidden.format, a.rows);
        if (a.hidden.format == MX_E2M1) {
            const int byte = mx_scale_byte<MX_E2M1>(m);
            const u32x2m c = mx_encode8<MX_E2M1>(v, byte);
            if (row_in && f < 4) reinterpret_cast<uint32_t*>(a.hidden.codes + at + strip / 2)[f] = c[0];
            if (row_in && f == 0) a.hidden.scales[(size_t)(tok0 + t) * mx_pitch(a.rows) + strip / 32] = (uint8_t)byte;
        } else {
            const int byte = mx_scale_byte<MX_E4M3>(m);
            const u32x2m c = mx_encode8<MX_E4M3>(v, byte);
            if (row_in && f < 4) reinterpret_cast<u32x2m*>(a.hidden.codes + at + strip)[f] = c;
            if (row_in && f == 0) a.hidden.scales[(size_t)(tok0 + t) * mx_pitch(a.rows) + strip / 32] = (uint8_t)byte;
        }
    }
}

template <int AF>
hipError_t few(const MxMatArgs& a, hipStream_t st) {
    const unsigned tg = (unsigned)((a.n + 15) / 16);
    if (a.gated)
        hipLaunchKernelGGL((mx_few_kernel<AF, true, 4>), dim3(tg * (unsigned)(a.rows / 32)), dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL((mx_few_kernel<AF, false, 1>), dim3(tg * (unsigned)((a.rows + 15) / 16)), dim3(512), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_matmul(const MxMatArgs& a, hipStream_t st) {
    if (a.n <= 0 || a.rows <= 0) return hipSuccess;
    // f32 sums of 8 bit codes: the bf16 MFMA's
    if (a.n > 16 && (a.gated || a.bf16 || a.act.format == MX_E2M1)) return launch_mx_tile(a, st);
    return a.act.format == MX_E2M1 ? few<MX_E2M1>(a, st) : few<MX_E4M3>(a, st);
}

}  // namespace dr
