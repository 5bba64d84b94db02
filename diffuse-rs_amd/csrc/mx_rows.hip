// mx_rows.hip -- microscaled rows made and read back: dr_mx_quantize,
// dr_mx_dequantize, dr_rms_norm_mx (the format: mx_common.hpp).
#include "mx_common.hpp"

namespace dr {
namespace {

// n / d for n < 2^31 (d == 1: m unused): m = ceil(2^(31 + s) / d), s = ceil(log2 d).
// (m d is less than 2^s over 2^(31 + s), and n times that less than 2^(31 + s): the quotient is exact.)
struct Div31 {
    uint32_t d, m, s;
    explicit Div31(uint32_t d_) : d(d_), m(0), s(0) {
        if (d == 1) return;
        while ((1ull << s) < d) ++s;
        m = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> (s - 1); }
};

// A lane holds 8 values, a quad of lanes a block: its largest magnitude is two
// lane exchanges away, and a row's codes leave in whole lines.  Both ways the bytes
// bound it: 18944 x 3584 bf16 to 4 bits 37 us (4.6 TB/s; a large copy reaches 4.8), back
// 26 us (its codes come from the memory-side cache).
template <int FMT, bool BF16>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const MxConvertArgs a, const Div31 by_blocks, uint32_t units) {
    const size_t pitch = (a.blocks + 3) / 4 * 4;
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    const bool live = u < units;  // (whole quads)
    const uint32_t b = (live ? u : 0) / 4, row = by_blocks(b), blk = b - row * a.blocks;
    float x[8];
    load8<BF16>(a.x, row * a.x_stride + (size_t)blk * 32 + (u & 3) * 8, x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    const int byte = mx_scale_byte<FMT>(quad_max(m));
    const u32x2m c = mx_encode8<FMT>(x, byte);
    if (!live) return;
    if constexpr (FMT == MX_E2M1)
        reinterpret_cast<uint32_t*>(a.rows.codes)[u] = c[0];
    else
        reinterpret_cast<u32x2m*>(a.rows.codes)[u] = c;
    if ((u & 3) == 0) a.rows.scales[row * pitch + blk] = (uint8_t)byte;
}

template <int FMT, bool BF16>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const MxConvertArgs a, const Div31 by_blocks, uint32_t units) {
    const size_t pitch = (a.blocks + 3) / 4 * 4;
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    if (u >= units) return;
    const uint32_t b = u / 4, row = by_blocks(b), blk = b - row * a.blocks;
    u32x2m c = {0, 0};
    if constexpr (FMT == MX_E2M1)
        c[0] = reinterpret_cast<const uint32_t*>(a.rows.codes)[u];
    else
        c = reinterpret_cast<const u32x2m*>(a.rows.codes)[u];
    float x[8];
    mx_decode8<FMT>(c, a.rows.scales[row * pitch + blk], x);
    store8<BF16>(a.out, (size_t)u * 8, x);
}

// The root of a row's mean square: sums of eight f32 squares are added in 64 bits
// (the reference adds f32 squares in 64 bits one by one), so that the factor is off by its own rounding alone:
// an f32 sum's few 2^-24 move ten times as many values past a border between codes.
template <int WAVES>
__device__ __forceinline__ float row_factor(double ss, double (&part)[WAVES], const MxNormArgs& a) {
#pragma unroll
    for (int d = 32; d; d >>= 1) ss += __shfl_xor(ss, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) ss += part[i];
    return (float)(1.0 / sqrt(ss / (double)a.cols + (double)a.eps));
}
__device__ __forceinline__ float squares8(const float (&h)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(h[i], h[i], s);
    return s;
}

// One workgroup per row; a row of up to 16384 values stays in registers between the
// sum and the codes, and the gain is on its way meanwhile.  8191 x 3584 bf16 with the
// residual 43 us (4.8 TB/s: the bytes bound it), one row of 4096 3.0 us (the launch
// and two trips to memory do).
template <int FMT, bool BF16, int NV>
__global__ __launch_bounds__(256) void mx_norm_kernel(const MxNormArgs a) {
    __shared__ double s_part[4];
    const size_t row = blockIdx.x;
    const size_t xo = row * a.x_stride, ro = row * (size_t)a.cols;
    float h[NV][8], w[NV][8];
    double ss = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * 256 + (int)threadIdx.x) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[v][i] = 0.0f, w[v][i] = 1.0f;
        if (at >= a.cols) continue;
        if (a.w) load8<false>(a.w, at, w[v]);  // (on its way while the squares are summed)
        load8<BF16>(a.x, xo + at, h[v]);
        if (a.residual) {
            float r[8];
            load8<BF16>(a.residual, ro + at, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[v][i] += r[i];
                if constexpr (BF16) h[v][i] = mx_f32(mx_bf16(h[v][i]));  // the stream is held in its type
            }
        }
        if (a.sum) store8<BF16>(a.sum, ro + at, h[v]);
        ss += squares8(h[v]);
    }
    const float scale = row_factor(ss, s_part, a);
    const size_t pitch = mx_pitch(a.cols), code_row = row * mx_row_bytes(FMT, a.cols);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * 256 + (int)threadIdx.x) * 8;
        float y[8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = h[v][i] * scale * w[v][i];
            m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
        }
        const int byte = mx_scale_byte<FMT>(quad_max(m));
        const u32x2m c = mx_encode8<FMT>(y, byte);
        if (at >= a.cols) continue;  // (whole quads)
        if constexpr (FMT == MX_E2M1)
            *reinterpret_cast<uint32_t*>(a.rows.codes + code_row + at / 2) = c[0];
        else
            *reinterpret_cast<u32x2m*>(a.rows.codes + code_row + at) = c;
        if ((threadIdx.x & 3) == 0) a.rows.scales[row * pitch + at / 32] = (uint8_t)byte;
    }
}

// Longer rows: twice over the row, the second time from the sum where there is
// one (it may lie over x or the residual).
template <int FMT, bool BF16>
__global__ __launch_bounds__(1024) void mx_norm_long_kernel(const MxNormArgs a) {
    __shared__ double s_part[16];
    const size_t row = blockIdx.x;
    const size_t xo = row * a.x_stride, ro = row * (size_t)a.cols;
    auto row8 = [&](int at, float (&h)[8]) {
        load8<BF16>(a.x, xo + at, h);
        if (!a.residual) return;
        float r[8];
        load8<BF16>(a.residual, ro + at, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] += r[i];
            if constexpr (BF16) h[i] = mx_f32(mx_bf16(h[i]));
        }
    };
    double ss = 0.0;
    for (int at = (int)threadIdx.x * 8; at < a.cols; at += 8192) {
        float h[8];
        row8(at, h);
        if (a.sum) store8<BF16>(a.sum, ro + at, h);
        ss += squares8(h);
    }
    const float scale = row_factor(ss, s_part, a);
    const size_t pitch = mx_pitch(a.cols), code_row = row * mx_row_bytes(FMT, a.cols);
    for (int at = (int)threadIdx.x * 8; at < a.cols; at += 8192) {
        float h[8], w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (a.sum)
            load8<BF16>(a.sum, ro + at, h);  // each thread's own values
        else
            row8(at, h);
        if (a.w) load8<false>(a.w, at, w);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = h[i] * scale * w[i];
            m = max(m, __float_as_uint(h[i]) & 0x7fffffffu);
        }
        const int byte = mx_scale_byte<FMT>(quad_max(m));
        const u32x2m c = mx_encode8<FMT>(h, byte);
        if constexpr (FMT == MX_E2M1)
            *reinterpret_cast<uint32_t*>(a.rows.codes + code_row + at / 2) = c[0];
        else
            *reinterpret_cast<u32x2m*>(a.rows.codes + code_row + at) = c;
        if ((threadIdx.x & 3) == 0) a.rows.scales[row * pitch + at / 32] = (uint8_t)byte;
    }
}

template <int FMT, bool BF16>
hipError_t norm(const MxNormArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)a.n), wg(256);
    if (a.cols <= 2048)
        hipLaunchKernelGGL((mx_norm_kernel<FMT, BF16, 1>), grid, wg, 0, st, a);
    else if (a.cols <= 4096)
        hipLaunchKernelGGL((mx_norm_kernel<FMT, BF16, 2>), grid, wg, 0, st, a);
    else if (a.cols <= 8192)
        hipLaunchKernelGGL((mx_norm_kernel<FMT, BF16, 4>), grid, wg, 0, st, a);
    else if (a.cols <= 16384)
        hipLaunchKernelGGL((mx_norm_kernel<FMT, BF16, 8>), grid, wg, 0, st, a);
    else
        hipLaunchKernelGGL((mx_norm_long_kernel<FMT, BF16>), grid, dim3(1024), 0, st, a);
    return hipGetLastError();
}

template <int FMT, bool BF16>
hipError_t convert(bool back, const MxConvertArgs& a, hipStream_t st) {
    const uint32_t units = a.n * a.blocks * 4;  // of 8 values
    if (units == 0) return hipSuccess;
    const dim3 grid((units - 1) / 256 + 1), wg(256);
    if (back)
        hipLaunchKernelGGL((mx_dequantize_kernel<FMT, BF16>), grid, wg, 0, st, a, Div31(a.blocks), units);
    else
        hipLaunchKernelGGL((mx_quantize_kernel<FMT, BF16>), grid, wg, 0, st, a, Div31(a.blocks), units);
    return hipGetLastError();
}

hipError_t convert(bool back, const MxConvertArgs& a, hipStream_t st) {
    if (a.rows.format == MX_E2M1) return a.bf16 ? convert<MX_E2M1, true>(back, a, st) : convert<MX_E2M1, false>(back, a, st);
    return a.bf16 ? convert<MX_E4M3, true>(back, a, st) : convert<MX_E4M3, false>(back, a, st);
}

}  // namespace

hipError_t launch_mx_quantize(const MxConvertArgs& a, hipStream_t st) { return convert(false, a, st); }
hipError_t launch_mx_dequantize(const MxConvertArgs& a, hipStream_t st) { return convert(true, a, st); }

hipError_t launch_mx_norm(const MxNormArgs& a, hipStream_t st) {
    if (a.n <= 0) return hipSuccess;
    if (a.rows.format == MX_E2M1) return a.bf16 ? norm<MX_E2M1, true>(a, st) : norm<MX_E2M1, false>(a, st);
    return a.bf16 ? norm<MX_E4M3, true>(a, st) : norm<MX_E4M3, false>(a, st);
}

}  // namespace dr
