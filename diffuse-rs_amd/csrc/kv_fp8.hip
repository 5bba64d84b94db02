// kv_fp8.hip -- store and gather of DR_PRECISION_FP8 cache layers: f32 rows ->
// e4m3 codes with a power-of-two scale per position and KV head (the format and
// the planes: fp8_common.hpp), and back to the f32 values that they stand for.
// Both are streams: 8 bytes of f32 rows (K and V) per value pair against 2 of
// codes, so HBM bounds the long calls and the launch the short ones.
//
// A row's values sit in one run of lanes, so its largest magnitude (and, with an
// epilogue, its sum of squares) is a few cross-lane steps.  Consecutive positions
// go by 32-position tiles, a workgroup per (tile, KV head, K or V): the codes
// turn through LDS into the plane's order and a tile is written whole, in 16-byte
// pieces.  A position list, and positions in too few tiles to occupy the CUs, go
// row by row, each run of lanes one row of K or V, straight between registers and
// the planes: K as the dwords of its 16-byte pieces, V as single bytes, which L2
// collects.
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
    static constexpr int RPT = 32 * LPR / NT;              // a tile's rows of a thread, consecutive: 4 or 8
    static constexpr int PER = NT / LPR;                   // rows of a workgroup, row by row
    static_assert(RPT % 4 == 0 && NV % 4 == 0, "V codes are packed four rows at a time, K codes four values");
    // LDS pitches: K's chunk of 32 x 16 bytes one 16-byte piece apart, so the
    // eight chunks that a wave writes sit on distinct banks; V's d-row of 32
    // codes at 48 bytes (two lanes to a bank, 16-byte aligned reads).
    static constexpr int KP = 32 * 16 + 16;
    static constexpr int VP = 48;
    static constexpr int LDS = HD / 16 * KP > HD * VP ? HD / 16 * KP : HD * VP;
};

// How a store or gather goes (pick_way, below).
enum Fp8Way { BY_TILES, BY_TILES_STREAM, BY_ROWS };

// The rows of workgroup block `blk`: row index r0 + i and position of entry i
// (0 .. PER - 1); consecutive positions are blocked at tile borders.
template <int PER>
struct Fp8Block {
    int r0, n, pos0;
    const int* pos;
    __device__ Fp8Block(int blk, int n_, int pos0_, const int* pos_) : n(n_), pos0(pos0_), pos(pos_) {
        r0 = pos0 >= 0 ? (pos0 / PER + blk) * PER - pos0 : blk * PER;
    }
    __device__ bool ok(int i) const { return r0 + i >= 0 && r0 + i < n; }
    __device__ int at(int i) const { return pos0 >= 0 ? pos0 + r0 + i : pos[r0 + i]; }
};

template <int HD, bool EPI, Fp8Way WAY>
__global__ __launch_bounds__(Fp8Rows<HD>::NT) void fp8_store_kernel(const StoreArgs a) {
    using G = Fp8Rows<HD>;
    constexpr bool ROWS = WAY == BY_ROWS;
    constexpr int RPT = ROWS ? 1 : G::RPT;
    __shared__ __align__(16) uint8_t tile[ROWS ? 16 : G::LDS];
    const bool isv = blockIdx.z != 0;
    const int g = blockIdx.y, tid = threadIdx.x;
    const int l = tid % G::LPR, i0 = tid / G::LPR * RPT;
    const Fp8Block<ROWS ? G::PER : 32> rows(blockIdx.x, a.n, a.pos0, a.pos);
    const float* src = (isv ? a.v : a.k) + (size_t)g * a.hd;
    // four consecutive values to a lane (a dword of K codes); V through LDS: values
    // LPR apart, so that the lanes' d-rows are neighbours there
    auto dim = [&](int i) { return isv && !ROWS ? l + G::LPR * i : (i / 4) * 4 * G::LPR + 4 * l + i % 4; };

    float x[RPT][G::NV];
    int pos[RPT];
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
        const bool ok = rows.ok(i0 + j);
        const float* row = src + (size_t)(ok ? rows.r0 + i0 + j : 0) * a.rstride;
        if ((ROWS || !isv) && a.vec) {
#pragma unroll
            for (int i = 0; i < G::NV; i += 4) {
                const f32x4* from = reinterpret_cast<const f32x4*>(row + dim(i));
                f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
                if (ok) t = WAY == BY_TILES_STREAM ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][i + e] = t[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < G::NV; ++i) {
                x[j][i] = 0.0f;
                if (ok && dim(i) < a.hd)
                    x[j][i] = WAY == BY_TILES_STREAM ? __builtin_nontemporal_load(row + dim(i)) : row[dim(i)];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < RPT; ++j) pos[j] = rows.ok(i0 + j) ? rows.at(i0 + j) : -1;

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
                for (int j = 0; j < RPT; ++j) x[j][i] += b;
            w[i] = !isv && a.kn_w && dim(i) < a.hd ? a.kn_w[dim(i)] : 1.0f;
        }
        if (norm) {
#pragma unroll
            for (int j = 0; j < RPT; ++j) {
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
            for (int j = 0; j < RPT; ++j) {
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
    for (int j = 0; j < RPT; ++j) {
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
    uint8_t* const kc = reinterpret_cast<uint8_t*>(a.kc);
    uint8_t* const vc = reinterpret_cast<uint8_t*>(a.vtc);
    if constexpr (ROWS) {
        if (pos[0] < 0) return;
        const size_t t = fp8_tile(g, a.cap, pos[0] / 32, HD);
        const int p = pos[0] % 32;
#pragma unroll
        for (int i = 0; i < G::NV; i += 4) {
            const int d = dim(i);
            const uint32_t w = fp8_pack4(x[0][i], x[0][i + 1], x[0][i + 2], x[0][i + 3]);
            if (!isv)
                *reinterpret_cast<uint32_t*>(kc + t + d / 16 * 512 + p * 16 + d % 16) = w;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) vc[t + (d + e) * 32 + p] = (uint8_t)(w >> (8 * e));
        }
        return;
    } else {
    if (!isv) {
#pragma unroll
        for (int j = 0; j < RPT; ++j)
#pragma unroll
            for (int i = 0; i < G::NV; i += 4) {
                const int d = dim(i);
                *reinterpret_cast<uint32_t*>(tile + d / 16 * G::KP + (i0 + j) * 16 + d % 16) =
                    fp8_pack4(x[j][i], x[j][i + 1], x[j][i + 2], x[j][i + 3]);
            }
    } else {
#pragma unroll
        for (int j = 0; j < RPT; j += 4)
#pragma unroll
            for (int i = 0; i < G::NV; ++i)
                *reinterpret_cast<uint32_t*>(tile + dim(i) * G::VP + i0 + j) =
                    fp8_pack4(x[j][i], x[j + 1][i], x[j + 2][i], x[j + 3][i]);
    }
    __syncthreads();
    // entry i is position i of the tile
    const size_t t = fp8_tile(g, a.cap, a.pos0 / 32 + blockIdx.x, HD);
    if (!isv) {
        for (int p = tid; p < HD / 16 * 32; p += G::NT)
            if (rows.ok(p % 32))
                *reinterpret_cast<u32x4*>(kc + t + p * 16) =
                    *reinterpret_cast<const u32x4*>(tile + p / 32 * G::KP + p % 32 * 16);
    } else {
        for (int p = tid; p < HD * 2; p += G::NT) {
            const int d = p / 2, i = p % 2 * 16;
            const uint8_t* from = tile + d * G::VP + i;
            uint8_t* to = vc + t + d * 32 + i;
            if (rows.ok(i) && rows.ok(i + 15)) {
                *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
            } else {
                for (int e = 0; e < 16; ++e)
                    if (rows.ok(i + e)) to[e] = from[e];
            }
        }
    }
    }
}

// The f32 values that the codes of the listed positions stand for.
template <int HD, bool ROWS>
__global__ __launch_bounds__(Fp8Rows<HD>::NT) void fp8_gather_kernel(const GatherArgs a) {
    using G = Fp8Rows<HD>;
    constexpr int RPT = ROWS ? 1 : G::RPT;
    __shared__ __align__(16) uint8_t tile[ROWS ? 16 : G::LDS];
    const bool isv = blockIdx.z != 0;
    const int g = blockIdx.y, tid = threadIdx.x;
    const int l = tid % G::LPR, i0 = tid / G::LPR * RPT;
    const Fp8Block<ROWS ? G::PER : 32> rows(blockIdx.x, a.n, a.pos0, a.pos);
    float scale[RPT];
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
        const int at = rows.ok(i0 + j) ? rows.at(i0 + j) : -1;
        scale[j] = at >= 0 ? fp8_scale(a.sc[fp8_scale_tile(g, a.cap, at / 32) + (isv ? 32 : 0) + at % 32]) : 0.0f;
    }
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(a.kc);
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(a.vtc);
    const size_t rstride = (size_t)a.n_head_kv * a.hd;
    float* const to = (isv ? a.out_v : a.out_k) + (size_t)g * a.hd;
    // four values from d on, of row r (written past the caches: 268 MB 78 -> 58
    // us, 256 x 32 rows of 128 4.1 -> 3.5)
    const bool vec = a.hd == HD && ((uintptr_t)to & 15) == 0;
    auto put4 = [&](int r, int d, uint32_t w, float f) __attribute__((always_inline)) {
        float* out = to + (size_t)r * rstride + d;
        const f32x4 y = {__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * f,
                         __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * f};
        if (vec) {
            __builtin_nontemporal_store(y, reinterpret_cast<f32x4*>(out));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < a.hd) out[e] = y[e];
        }
    };
    if constexpr (ROWS) {
        if (!rows.ok(i0)) return;
        const int at = rows.at(i0), p = at % 32;
        const size_t t = fp8_tile(g, a.cap, at / 32, HD);
        uint32_t w[G::NV / 4];
#pragma unroll
        for (int i = 0; i < G::NV / 4; ++i) {
            const int d = (i * G::LPR + l) * 4;
            if (!isv) {
                w[i] = *reinterpret_cast<const uint32_t*>(kc + t + d / 16 * 512 + p * 16 + d % 16);
            } else {
                uint32_t b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = vc[t + (d + e) * 32 + p];
                w[i] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
            }
        }
#pragma unroll
        for (int i = 0; i < G::NV / 4; ++i) put4(rows.r0 + i0, (i * G::LPR + l) * 4, w[i], scale[0]);
    } else {
        // (a tile lies within the plane whole, whatever part of it was asked for)
        const size_t t = fp8_tile(g, a.cap, a.pos0 / 32 + blockIdx.x, HD);
        for (int p = tid; p < HD * 2; p += G::NT) {
            uint8_t* lds = isv ? tile + p / 2 * G::VP + p % 2 * 16 : tile + p / 32 * G::KP + p % 32 * 16;
            *reinterpret_cast<u32x4*>(lds) = *reinterpret_cast<const u32x4*>((isv ? vc : kc) + t + p * 16);
        }
        __syncthreads();
        if (!isv) {
#pragma unroll
            for (int j = 0; j < RPT; ++j)
                if (rows.ok(i0 + j))
#pragma unroll
                    for (int i = 0; i < G::NV / 4; ++i) {
                        const int d = (i * G::LPR + l) * 4;
                        put4(rows.r0 + i0 + j, d,
                             *reinterpret_cast<const uint32_t*>(tile + d / 16 * G::KP + (i0 + j) * 16 + d % 16),
                             scale[j]);
                    }
        } else {
#pragma unroll
            for (int j = 0; j < RPT; j += 4)
#pragma unroll
                for (int i = 0; i < G::NV; ++i) {
                    const int d = l + G::LPR * i;
                    if (d >= a.hd) continue;
                    const int w = *reinterpret_cast<const int*>(tile + d * G::VP + i0 + j);
                    const float y[4] = {__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1),
                                        __builtin_amdgcn_cvt_f32_fp8(w, 2), __builtin_amdgcn_cvt_f32_fp8(w, 3)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (rows.ok(i0 + j + e)) __builtin_nontemporal_store(y[e] * scale[j + e], to + (size_t)(rows.r0 + i0 + j + e) * rstride + d);
                }
        }
    }
}

// Workgroups along the rows, of PER rows each: consecutive positions are blocked
// at multiples of PER.
int fp8_blocks(int n, int pos0, int per) {
    return pos0 >= 0 ? (pos0 + n - 1) / per - pos0 / per + 1 : (n + per - 1) / per;
}

// Row by row: every position list; consecutive positions where their tiles give
// fewer workgroups than a CU each (2 heads of 512, 256 rows, store / gather: by
// tiles 8.6 / 6.1 us, by rows 4.0 / 3.4; 32 heads of 128, 256 rows, a list that
// could go no other way: 6.8 / 4.9 against 4.5 / 3.5 by tiles).  A store whose
// rows no cache level holds reads past them (32768 rows x 8 heads of 128, 268 MB:
// 71 -> 64 us; where L2 or the memory-side cache may still hold them, 256 x 32
// heads: 4.6 -> 5.5, 8192 x 8: 17.8 -> 19.3).
Fp8Way pick_way(int n, int pos0, int n_head_kv, int hd, int n_cu) {
    if (pos0 < 0 || (long)fp8_blocks(n, pos0, 32) * n_head_kv * 2 < n_cu) return BY_ROWS;
    return (long)n * n_head_kv * hd >= 16L << 20 ? BY_TILES_STREAM : BY_TILES;
}

template <int HD, Fp8Way WAY>
hipError_t store(const StoreArgs& a, hipStream_t st) {
    const int per = WAY == BY_ROWS ? Fp8Rows<HD>::PER : 32;
    const dim3 grid((unsigned)fp8_blocks(a.n, a.pos0, per), (unsigned)a.n_head_kv, 2);
    if (a.kn_w || a.kb || a.vb || a.v_norm || a.rope)
        hipLaunchKernelGGL((fp8_store_kernel<HD, true, WAY>), grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    else
        hipLaunchKernelGGL((fp8_store_kernel<HD, false, WAY>), grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t store(const StoreArgs& a, hipStream_t st) {
    switch (pick_way(a.n, a.pos0, a.n_head_kv, a.hd, a.n_cu)) {
        case BY_ROWS: return store<HD, BY_ROWS>(a, st);
        case BY_TILES_STREAM: return store<HD, BY_TILES_STREAM>(a, st);
        default: return store<HD, BY_TILES>(a, st);
    }
}

template <int HD, bool ROWS>
hipError_t gather(const GatherArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)fp8_blocks(a.n, a.pos0, ROWS ? Fp8Rows<HD>::PER : 32), (unsigned)a.n_head_kv, 2);
    hipLaunchKernelGGL((fp8_gather_kernel<HD, ROWS>), grid, dim3(Fp8Rows<HD>::NT), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_store_fp8(int hd_tile, const StoreArgs& a, hipStream_t st) {
    if (a.n <= 0) return hipSuccess;
    if (!a.sc || a.rstride < a.n_head_kv * a.hd || (a.pos0 < 0 && !a.pos)) return hipErrorInvalidValue;
    switch (hd_tile) {
        case 64: return store<64>(a, st);
        case 128: return store<128>(a, st);
        case 256: return store<256>(a, st);
        case 512: return store<512>(a, st);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_gather_fp8(int hd_tile, const GatherArgs& a, hipStream_t st) {
    if (a.n <= 0) return hipSuccess;
    if (!a.sc || (a.pos0 < 0 && !a.pos)) return hipErrorInvalidValue;
    const bool rows = pick_way(a.n, a.pos0, a.n_head_kv, a.hd, a.n_cu) == BY_ROWS;
    switch (hd_tile) {
        case 64: return rows ? gather<64, true>(a, st) : gather<64, false>(a, st);
        case 128: return rows ? gather<128, true>(a, st) : gather<128, false>(a, st);
        case 256: return rows ? gather<256, true>(a, st) : gather<256, false>(a, st);
        case 512: return rows ? gather<512, true>(a, st) : gather<512, false>(a, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dr
