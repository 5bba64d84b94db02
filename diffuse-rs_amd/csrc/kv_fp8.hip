// kv_fp8.hip -- store and gather of DR_PRECISION_FP8 cache layers: f32 rows ->
// e4m3 codes with a power-of-two scale per position and KV head (the format and
// the planes: fp8_common.hpp), and back to the f32 values that they stand for.
// Both are streams: 8 bytes of f32 rows (K and V) per value pair against 2 of
// codes, so HBM bounds the long calls and the launch the short ones.
//
// One workgroup per (32 rows, KV head, K or V).  A row's values sit in one run
// of lanes, so its largest magnitude (and, with an epilogue, its sum of
// squares) is a few cross-lane steps; the codes turn through LDS into the
// plane's order and leave as 16-byte pieces.  Rows of consecutive positions
// are blocked at 32-position tiles, which are then written whole; a position
// list is blocked by 32 entries, and its V codes leave as dwords where four
// aligned neighbours are in the block, as bytes elsewhere.
#include <algorithm>

#include "fp8_common.hpp"

#include <math.h>

namespace dr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// RoPE's rotation of one pair (ops.rs:447-448), without fused multiply-adds
// as Rust evaluates it.
__device__ __forceinline__ float rope_lo(float a, float b, float sn, float cs) {
#pragma clang fp contract(off)
    return a * cs - b * sn;
}
__device__ __forceinline__ float rope_hi(float a, float b, float sn, float cs) {
#pragma clang fp contract(off)
    return a * sn + b * cs;
}

template <int HD>
struct Fp8Rows {
    static constexpr int LPR = HD / 4 < 64 ? HD / 4 : 64;  // lanes of a row
    static constexpr int NV = HD / LPR;                    // values of a row in a lane
    static constexpr int NT = HD < 128 ? 128 : 256;        // threads
    static constexpr int RPT = 32 * LPR / NT;              // rows of a thread, consecutive: 4 or 8
    static_assert(RPT % 4 == 0 && NV % 4 == 0, "V codes are packed four rows at a time, K codes four values");
    // LDS pitches: K's chunk of 32 x 16 bytes one 16-byte piece apart, so the
    // eight chunks that a wave writes sit on distinct banks; V's d-row of 32
    // codes at 48 bytes (two lanes to a bank, 16-byte aligned reads).
    static constexpr int KP = 32 * 16 + 16;
    static constexpr int VP = 48;
    static constexpr int LDS = HD / 16 * KP > HD * VP ? HD / 16 * KP : HD * VP;
};

// The rows of workgroup block `blk`: row index r0 + i and position of entry i
// (0..31); consecutive positions are blocked at tile borders.
struct Fp8Block {
    int r0, n, pos0;
    const int* pos;
    __device__ Fp8Block(int blk, int n_, int pos0_, const int* pos_) : n(n_), pos0(pos0_), pos(pos_) {
        r0 = pos0 >= 0 ? (pos0 / 32 + blk) * 32 - pos0 : blk * 32;
    }
    __device__ bool ok(int i) const { return r0 + i >= 0 && r0 + i < n; }
    __device__ int at(int i) const { return pos0 >= 0 ? pos0 + r0 + i : pos[r0 + i]; }
};

// Position list: the groups of entries whose positions share an aligned four
// (entry of the first, how many, position of the first), for dword accesses
// of V's d-rows.  Wave 0; entries past the list's end are in no group.
struct Fp8Groups {
    int n;
    int first[32], count[32], pos[32];
};
__device__ __forceinline__ void fp8_groups(const Fp8Block& rows, Fp8Groups& gr) {
    if (threadIdx.x < 64) {
        const int i = threadIdx.x;
        const bool ok = i < 32 && rows.ok(i);
        const int p = ok ? rows.at(i) : -1;
        const int prev = __shfl_up(p, 1);
        const bool head = ok && (i == 0 || (prev >> 2) != (p >> 2));
        const uint64_t heads = __ballot(head);
        const int total = __popcll(__ballot(ok));
        if (head) {
            const int k = __popcll(heads & ((1ull << i) - 1));
            const uint64_t later = i < 63 ? heads >> (i + 1) : 0;
            gr.first[k] = i;
            gr.count[k] = (later ? i + 1 + (int)__builtin_ctzll(later) : total) - i;
            gr.pos[k] = p;
        }
        if (i == 0) gr.n = __popcll(heads);
    }
}

template <int HD, bool EPI>
__global__ __launch_bounds__(Fp8Rows<HD>::NT) void fp8_store_kernel(const StoreArgs a) {
    using G = Fp8Rows<HD>;
    __shared__ __align__(16) uint8_t tile[G::LDS];
    __shared__ Fp8Groups groups;
    const bool isv = blockIdx.z != 0;
    const int g = blockIdx.y, tid = threadIdx.x;
    const int l = tid % G::LPR, i0 = tid / G::LPR * G::RPT;
    const Fp8Block rows(blockIdx.x, a.n, a.pos0, a.pos);
    const float* src = (isv ? a.v : a.k) + (size_t)g * a.hd;
    // K: four consecutive values to a lane (a dword of codes); V: values LPR
    // apart, so that the lanes' d-rows are neighbours in LDS
    auto dim = [&](int i) { return isv ? l + G::LPR * i : (i / 4) * 4 * G::LPR + 4 * l + i % 4; };

    float x[G::RPT][G::NV];
    int pos[G::RPT];
#pragma unroll
    for (int j = 0; j < G::RPT; ++j) {
        const bool ok = rows.ok(i0 + j);
        const float* row = src + (size_t)(ok ? rows.r0 + i0 + j : 0) * a.rstride;
        if (!isv && a.vec) {
#pragma unroll
            for (int i = 0; i < G::NV; i += 4) {
                const f32x4 t = ok ? *reinterpret_cast<const f32x4*>(row + dim(i)) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][i + e] = t[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < G::NV; ++i) x[j][i] = ok && dim(i) < a.hd ? row[dim(i)] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < G::RPT; ++j) pos[j] = rows.ok(i0 + j) ? rows.at(i0 + j) : -1;

    if constexpr (EPI) {
        // the K / V part of the Q/K/V epilogue (forward.rs:291-310) in the
        // order of dr_qkv_epilogue: bias, RMSNorm (f32 squares summed in f64;
        // K's gain, none for V), RoPE of K
        const float* bias = isv ? a.vb : a.kb;
        const bool norm = isv ? a.v_norm != 0 : a.kn_w != nullptr;
        float w[G::NV];
#pragma unroll
        for (int i = 0; i < G::NV; ++i) {
            const float b = bias && dim(i) < a.hd ? bias[(size_t)g * a.hd + dim(i)] : 0.0f;
            if (bias)
#pragma unroll
                for (int j = 0; j < G::RPT; ++j) x[j][i] += b;
            w[i] = !isv && a.kn_w && dim(i) < a.hd ? a.kn_w[dim(i)] : 1.0f;
        }
        if (norm) {
#pragma unroll
            for (int j = 0; j < G::RPT; ++j) {
                double ss = 0.0;
#pragma unroll
                for (int i = 0; i < G::NV; ++i) {
                    const float sq = x[j][i] * x[j][i];
                    ss += (double)sq;
                }
#pragma unroll
                for (int off = G::LPR / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
                const float sc = 1.0f / (float)sqrt(ss / (double)a.hd + (double)a.kn_eps);
#pragma unroll
                for (int i = 0; i < G::NV; ++i) x[j][i] = isv ? x[j][i] * sc : x[j][i] * sc * w[i];
            }
        }
        if (!isv && a.rope) {
            // a dim's partner (d +- rot/2, rot/2 a multiple of 4) is the same
            // element of another four of the row
            const int half = a.rot / 2;
#pragma unroll
            for (int j = 0; j < G::RPT; ++j) {
                float y[G::NV];
#pragma unroll
                for (int i = 0; i < G::NV; ++i) {
                    const int d = dim(i), pd = d < half ? d + half : d - half;
                    const int quad = (d < a.rot ? pd : d) / 4;
                    const int from = (tid & 63) / G::LPR * G::LPR + quad % G::LPR;
                    float xp = 0.0f;
#pragma unroll
                    for (int c = 0; c < G::NV / 4; ++c) {
                        const float t = __shfl(x[j][4 * c + i % 4], from);
                        if (quad / G::LPR == c) xp = t;
                    }
                    y[i] = x[j][i];
                    if (d < a.rot && pos[j] >= 0) {
                        const float2 t = *reinterpret_cast<const float2*>(
                            a.rope + ((size_t)pos[j] * half + (d < half ? d : pd)) * 2);
                        y[i] = d < half ? rope_lo(x[j][i], xp, t.x, t.y) : rope_hi(xp, x[j][i], t.x, t.y);
                    }
                }
#pragma unroll
                for (int i = 0; i < G::NV; ++i) x[j][i] = y[i];
            }
        }
    }

    // each row's scale, and its values divided by it
#pragma unroll
    for (int j = 0; j < G::RPT; ++j) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < G::NV; ++i) top = max(top, __float_as_uint(x[j][i]) & 0x7fffffffu);
#pragma unroll
        for (int off = G::LPR / 2; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
        const int byte = fp8_scale_byte(top);
        const float inv = byte == FP8_NAN ? 0.0f : fp8_inverse(byte);
#pragma unroll
        for (int i = 0; i < G::NV; ++i) x[j][i] = byte == FP8_NAN ? 0.0f : x[j][i] * inv;
        if (l == 0 && pos[j] >= 0)
            a.sc[fp8_scale_tile(g, a.cap, pos[j] / 32) + (isv ? 32 : 0) + pos[j] % 32] = (uint8_t)byte;
    }
    if (!isv) {
#pragma unroll
        for (int j = 0; j < G::RPT; ++j)
#pragma unroll
            for (int i = 0; i < G::NV; i += 4) {
                const int d = dim(i);
                *reinterpret_cast<uint32_t*>(tile + d / 16 * G::KP + (i0 + j) * 16 + d % 16) =
                    fp8_pack4(x[j][i], x[j][i + 1], x[j][i + 2], x[j][i + 3]);
            }
    } else {
#pragma unroll
        for (int j = 0; j < G::RPT; j += 4)
#pragma unroll
            for (int i = 0; i < G::NV; ++i)
                *reinterpret_cast<uint32_t*>(tile + dim(i) * G::VP + i0 + j) =
                    fp8_pack4(x[j][i], x[j + 1][i], x[j + 2][i], x[j + 3][i]);
        if (a.pos0 < 0) fp8_groups(rows, groups);
    }
    __syncthreads();

    if (!isv) {
        uint8_t* kc = reinterpret_cast<uint8_t*>(a.kc);
        for (int p = tid; p < HD / 16 * 32; p += G::NT) {
            const int c = p / 32, i = p % 32;
            if (!rows.ok(i)) continue;
            const int at = rows.at(i);
            *reinterpret_cast<u32x4*>(kc + fp8_tile(g, a.cap, at / 32, HD) + c * 512 + at % 32 * 16) =
                *reinterpret_cast<const u32x4*>(tile + c * G::KP + i * 16);
        }
    } else if (a.pos0 >= 0) {
        // entry i is position i of the tile
        uint8_t* vt = reinterpret_cast<uint8_t*>(a.vtc) + fp8_tile(g, a.cap, a.pos0 / 32 + blockIdx.x, HD);
        for (int p = tid; p < HD * 2; p += G::NT) {
            const int d = p / 2, i = p % 2 * 16;
            const uint8_t* from = tile + d * G::VP + i;
            uint8_t* to = vt + d * 32 + i;
            if (rows.ok(i) && rows.ok(i + 15)) {
                *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
            } else {
                for (int e = 0; e < 16; ++e)
                    if (rows.ok(i + e)) to[e] = from[e];
            }
        }
    } else {
        uint8_t* vt = reinterpret_cast<uint8_t*>(a.vtc);
        for (int p = tid; p < HD * groups.n; p += G::NT) {
            const int d = p / groups.n, k = p - d * groups.n;
            const int first = groups.first[k], count = groups.count[k], at = groups.pos[k];
            const uint8_t* from = tile + d * G::VP + first;
            uint8_t* to = vt + fp8_tile(g, a.cap, at / 32, HD) + d * 32 + at % 32;
            if (count == 4) {
                *reinterpret_cast<uint32_t*>(to) =
                    from[0] | (uint32_t)from[1] << 8 | (uint32_t)from[2] << 16 | (uint32_t)from[3] << 24;
            } else {
                // (positions of a group ascend but may skip some of the four)
                for (int e = 0; e < count; ++e) to[rows.at(first + e) - at] = from[e];
            }
        }
    }
}

// The f32 values that the codes of the listed positions stand for.
template <int HD>
__global__ __launch_bounds__(Fp8Rows<HD>::NT) void fp8_gather_kernel(const GatherArgs a) {
    using G = Fp8Rows<HD>;
    __shared__ __align__(16) uint8_t tile[G::LDS];
    const bool isv = blockIdx.z != 0;
    const int g = blockIdx.y, tid = threadIdx.x;
    const int l = tid % G::LPR, i0 = tid / G::LPR * G::RPT;
    const Fp8Block rows(blockIdx.x, a.n, a.pos0, a.pos);
    float scale[G::RPT];
#pragma unroll
    for (int j = 0; j < G::RPT; ++j) {
        const int at = rows.ok(i0 + j) ? rows.at(i0 + j) : -1;
        scale[j] = at >= 0 ? fp8_scale(a.sc[fp8_scale_tile(g, a.cap, at / 32) + (isv ? 32 : 0) + at % 32]) : 0.0f;
    }
    if (!isv) {
        const uint8_t* kc = reinterpret_cast<const uint8_t*>(a.kc);
        for (int p = tid; p < HD / 16 * 32; p += G::NT) {
            const int c = p / 32, i = p % 32;
            if (!rows.ok(i)) continue;
            const int at = rows.at(i);
            *reinterpret_cast<u32x4*>(tile + c * G::KP + i * 16) =
                *reinterpret_cast<const u32x4*>(kc + fp8_tile(g, a.cap, at / 32, HD) + c * 512 + at % 32 * 16);
        }
    } else if (a.pos0 >= 0) {
        // (a tile lies within the plane whole, whatever part of it was asked for)
        const uint8_t* vt =
            reinterpret_cast<const uint8_t*>(a.vtc) + fp8_tile(g, a.cap, a.pos0 / 32 + blockIdx.x, HD);
        for (int p = tid; p < HD * 2; p += G::NT)
            *reinterpret_cast<u32x4*>(tile + p / 2 * G::VP + p % 2 * 16) =
                *reinterpret_cast<const u32x4*>(vt + p * 16);
    } else {
        const uint8_t* vt = reinterpret_cast<const uint8_t*>(a.vtc);
        for (int p = tid; p < HD * 32; p += G::NT) {
            const int d = p / 32, i = p % 32;
            if (!rows.ok(i)) continue;
            const int at = rows.at(i);
            tile[d * G::VP + i] = vt[fp8_tile(g, a.cap, at / 32, HD) + d * 32 + at % 32];
        }
    }
    __syncthreads();
    const size_t rstride = (size_t)a.n_head_kv * a.hd;
    if (!isv) {
        const bool vec = a.hd == HD && ((uintptr_t)a.out_k & 15) == 0;
#pragma unroll
        for (int j = 0; j < G::RPT; ++j) {
            if (!rows.ok(i0 + j)) continue;
            float* out = a.out_k + (size_t)(rows.r0 + i0 + j) * rstride + (size_t)g * a.hd;
#pragma unroll
            for (int i = 0; i < G::NV; i += 4) {
                const int d = (i / 4) * 4 * G::LPR + 4 * l;
                const int w = *reinterpret_cast<const int*>(tile + d / 16 * G::KP + (i0 + j) * 16 + d % 16);
                const f32x4 y = {__builtin_amdgcn_cvt_f32_fp8(w, 0) * scale[j],
                                 __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale[j],
                                 __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale[j],
                                 __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale[j]};
                if (vec) {
                    *reinterpret_cast<f32x4*>(out + d) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < a.hd) out[d + e] = y[e];
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < G::RPT; j += 4)
#pragma unroll
            for (int i = 0; i < G::NV; ++i) {
                const int d = l + G::LPR * i;
                if (d >= a.hd) continue;
                const int w = *reinterpret_cast<const int*>(tile + d * G::VP + i0 + j);
                const float y[4] = {__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1),
                                    __builtin_amdgcn_cvt_f32_fp8(w, 2), __builtin_amdgcn_cvt_f32_fp8(w, 3)};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (rows.ok(i0 + j + e))
                        a.out_v[(size_t)(rows.r0 + i0 + j + e) * rstride + (size_t)g * a.hd + d] =
                            y[e] * scale[j + e];
            }
    }
}

// Workgroups along the rows: tiles that consecutive positions touch, or
// blocks of 32 list entries.
int fp8_blocks(int n, int pos0) { return pos0 >= 0 ? (pos0 + n - 1) / 32 - pos0 / 32 + 1 : (n + 31) / 32; }

template <int HD>
hipError_t store(const StoreArgs& a, bool epi, hipStream_t st) {
    const dim3 grid((unsigned)fp8_blocks(a.n, a.pos0), (unsigned)a.n_head_kv, 2);
    if (epi)
        hipLaunchKernelGGL((fp8_store_kernel<HD, true>), grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    else
        hipLaunchKernelGGL((fp8_store_kernel<HD, false>), grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t gather(const GatherArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)fp8_blocks(a.n, a.pos0), (unsigned)a.n_head_kv, 2);
    hipLaunchKernelGGL(fp8_gather_kernel<HD>, grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_store_fp8(int hd_tile, const StoreArgs& a, hipStream_t st) {
    if (a.n <= 0) return hipSuccess;
    if (!a.sc || a.rstride < a.n_head_kv * a.hd || (a.pos0 < 0 && !a.pos)) return hipErrorInvalidValue;
    const bool epi = a.kn_w || a.kb || a.vb || a.v_norm || a.rope;
    switch (hd_tile) {
        case 64: return store<64>(a, epi, st);
        case 128: return store<128>(a, epi, st);
        case 256: return store<256>(a, epi, st);
        case 512: return store<512>(a, epi, st);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_gather_fp8(int hd_tile, const GatherArgs& a, hipStream_t st) {
    if (a.n <= 0) return hipSuccess;
    if (!a.sc || (a.pos0 < 0 && !a.pos)) return hipErrorInvalidValue;
    switch (hd_tile) {
        case 64: return gather<64>(a, st);
        case 128: return gather<128>(a, st);
        case 256: return gather<256>(a, st);
        case 512: return gather<512>(a, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dr
