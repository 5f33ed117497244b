// gfx950 causal attention of many rows over paged caches in float32: what
// rows_kernels.hip, which describes both, does not take on 16-bit products.
#include "rows_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

// Everything in float32: 32 columns a wavefront on v_mfma_f32_32x32x2_f32, the
// products of cross_attend_f32_kernel. Cache values of any type are widened
// (codes times their scales) on their way into LDS.
template <int CT, int D, bool FULL>
__global__ __launch_bounds__(64 * kRWaves, D == 256 ? 1 : 2) void rows_attend_f32_kernel(RowsArgs a, int col_tiles) {
    constexpr int kKeys = D == 64 ? 64 : 32;   // keys a tile
    constexpr int kBytes = kKeys * D * 4;
    constexpr int kSize = CT == 0 ? 4 : CT <= 2 ? 2 : 1;
    constexpr int kPer = 16 / kSize;           // values of a 16-byte piece of a cache row
    constexpr int kRowPieces = D / kPer;
    constexpr int kStage = (kKeys * kRowPieces + 255) / 256;  // pieces a thread stages
    extern __shared__ __align__(16) unsigned char smem[];  // [2][keys, values]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    constexpr int kWgCols = kRWaves * 32;
    const RowsPlace p = rows_place<kKeys>(a, col_tiles, kWgCols);
    if (!p.ok) return;
    const int col0 = p.ct * kWgCols + wave * 32;
    const bool live = col0 < p.cols;
    const int first = p.pos + min(col0, p.cols - 1) / a.group, last = p.pos + (min(col0 + 32, p.cols) - 1) / a.group;
    const int at = p.pos + min(col0 + n, p.cols - 1) / a.group;
    const unsigned char *kp = a.c.k + static_cast<long long>(p.h) * a.k_head;
    const unsigned char *vp = a.c.v + static_cast<long long>(p.h) * a.v_head;

    auto rows_of = [&](int i) { return pool_row(a, p.b, min(tile_key<kKeys>(p, i) + (lane & (kKeys - 1)), p.end - 1)); };
    uint4 kst[kStage], vst[kStage];
    float kss[kStage], vss[kStage];
    auto fetch = [&](int rows) {
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kRowPieces, c = piece % kRowPieces;
            const long long src = __shfl(rows, row & (kKeys - 1));
            const bool in = row < kKeys;
            kst[k] = in && (FULL || c * kPer < a.c.qk) ? *reinterpret_cast<const uint4 *>(kp + src * a.k_row + c * 16) : make_uint4(0, 0, 0, 0);
            vst[k] = in && (FULL || c * kPer < a.c.vd) ? *reinterpret_cast<const uint4 *>(vp + src * a.v_row + c * 16) : make_uint4(0, 0, 0, 0);
            if constexpr (CT >= 3) {
                const long long sat = (src >> a.c.sshift) * a.c.kv_heads + p.h;
                kss[k] = a.c.ks[sat];
                vss[k] = a.c.vs[sat];
            }
        }
    };
    auto widen = [&](const uint4 &v, int e, float sc) {  // value e of a piece
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (CT == 0) return __uint_as_float(w[e]);
        if constexpr (CT == 1 || CT == 2) return half_value(static_cast<uint16_t>(w[(e >> 1) & 3] >> (16 * (e & 1))), CT);
        if constexpr (CT == 3) return static_cast<float>(static_cast<int32_t>(w[(e >> 2) & 3] << (24 - 8 * (e & 3))) >> 24) * sc;
        const int x = static_cast<int>(w[(e >> 2) & 3] >> (8 * (e & 3)));
        return __builtin_amdgcn_cvt_f32_fp8(x, 0) * sc;
    };
    auto store = [&](int j, int buf) {
        unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kRowPieces, c = piece % kRowPieces;
            if (row >= kKeys) continue;
            const bool dead = j + row >= p.end;  // values behind the last key: 0
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
                const int c4 = c * (kPer / 4) + e / 4;  // 16-byte piece of the float32 row
                *reinterpret_cast<float4 *>(kt + row * D * 4 + ((c4 ^ (row & 15)) * 16)) =
                    make_float4(widen(kst[k], e, kss[k]), widen(kst[k], e + 1, kss[k]), widen(kst[k], e + 2, kss[k]), widen(kst[k], e + 3, kss[k]));
                *reinterpret_cast<float4 *>(vt + row * D * 4 + ((c4 ^ (((row >> 2) & 1) << 3)) * 16)) =
                    dead ? make_float4(0, 0, 0, 0)
                         : make_float4(widen(vst[k], e, vss[k]), widen(vst[k], e + 1, vss[k]), widen(vst[k], e + 2, vss[k]),
                                       widen(vst[k], e + 3, vss[k]));
            }
        }
    };

    // The queries: lane (n, half) holds coordinates 8 s + 4 half + 0..3 of its column.
    float q[D / 2];
    {
        const int col = min(col0 + n, p.cols - 1);
        const long long qo = static_cast<long long>(p.b) * a.q_stream + static_cast<long long>(col / a.group) * a.q_row +
                             static_cast<long long>(p.h * a.group + col % a.group) * a.c.qk;
#pragma unroll
        for (int s = 0; s < D / 8; ++s) {
            const int d = 8 * s + 4 * half;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[4 * s + e] = 0.0f;
            if (FULL || d < a.c.qk) {
                if (a.type == 0 && (a.aligned & 1)) {
                    const float4 y = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + qo + d);
                    q[4 * s] = y.x, q[4 * s + 1] = y.y, q[4 * s + 2] = y.z, q[4 * s + 3] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[4 * s + e] = load_any(a.q, a.type, qo + d + e);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) q[4 * s + e] *= a.scale_log2;
        }
    }
    f32x16 o[D / 32];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[v][e] = 0.0f;

    int rows = 0;
    if (p.i0 < p.i1) {
        rows = rows_of(p.i0);
        fetch(rows);
        store(tile_key<kKeys>(p, p.i0), 0);
        if (p.i0 + 1 < p.i1) rows = rows_of(p.i0 + 1);
    }
    int buf = 0;
    for (int i = p.i0; i < p.i1; ++i, buf ^= 1) {
        const int j = tile_key<kKeys>(p, i);
        __syncthreads();  // this tile is whole, and the other buffer's readers are done
        const bool more = i + 1 < p.i1;
        if (more) {
            fetch(rows);
            if (i + 2 < p.i1) rows = rows_of(i + 2);
        }
        const unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
#pragma unroll
        for (int kb = 0; kb < kKeys / 32; ++kb) {
            const int j0 = j + 32 * kb;
            if (!live || none_sees(a, first, last, j0, j0 + 31)) continue;
            f32x16 s;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
            const unsigned char *kr = kt + (32 * kb + n) * D * 4;
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
                if (FULL || 8 * c < a.c.qk) {
                    const float4 ka = *reinterpret_cast<const float4 *>(kr + ((2 * c + half) ^ (n & 15)) * 16);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.x, q[4 * c], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.y, q[4 * c + 1], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.z, q[4 * c + 2], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.w, q[4 * c + 3], s, 0, 0, 0);
                }
            if (!all_see(a, first, last, j0, j0 + 31)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = sees(a, at, j0 + 8 * (e >> 2) + 4 * half + (e & 3)) ? s[e] : -INFINITY;
            }
            float mt = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mt = fmaxf(mt, s[e]);
            mt = halves_max(mt);
            if (__any(mt > m + 8.0f)) {
                const float mn = fmaxf(m, mt);
                const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int v = 0; v < D / 32; ++v) o[v] *= f;
            }
            const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e] - mu);
                l += s[e];
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3);
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    if (FULL || 32 * v < a.c.vd) {
                        const float va = *reinterpret_cast<const float *>(vt + row * D * 4 + (((32 * v + n) * 4) ^ (half << 7)));
                        o[v] = __builtin_amdgcn_mfma_f32_32x32x2f32(va, s[e], o[v], 0, 0, 0);
                    }
            }
        }
        if (more) store(tile_key<kKeys>(p, i + 1), buf ^ 1);
    }
    if (!live) return;
    const float sum = halves_sum(l);
    const int col = col0 + n;
    bool nan = false;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) nan |= o[v][e] != o[v][e];
    if (col < p.cols) {
        const int head = p.h * a.group + col % a.group, row = col / a.group;
        const long long pi = ((static_cast<long long>(p.b) * a.t + row) * a.heads + head) * a.splits + p.sp;
        const long long to = a.part ? pi * a.c.vd
                                    : static_cast<long long>(p.b) * a.out_stream + static_cast<long long>(row) * a.out_row +
                                          static_cast<long long>(head) * a.c.vd;
        const float f = a.part ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int v = 0; v < D / 32; ++v)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 32 * v + 8 * (e >> 2) + 4 * half + (e & 3);
                if (FULL || d < a.c.vd) store_any(a.part ? a.part : a.out, a.part ? 0 : a.type, to + d, o[v][e] * f);
            }
        if (a.part && half == 0) {
            a.part_ml[2 * pi] = m;
            a.part_ml[2 * pi + 1] = sum;
        }
    }
    const unsigned long long bad = __ballot(nan && col < p.cols);
    if (bad) repair_columns<kKeys>(a, p, col0, static_cast<unsigned>(bad) | static_cast<unsigned>(bad >> 32));
}

template <int CT, int D>
hipError_t launch_f32_full(const RowsArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> full{0}, part{0};
    constexpr int lds = 4 * (D == 64 ? 64 : 32) * D * 4;
    return a.c.qk == D && a.c.vd == D ? launch_with(&rows_attend_f32_kernel<CT, D, true>, a, kRWaves * 32, lds, full, s)
                                      : launch_with(&rows_attend_f32_kernel<CT, D, false>, a, kRWaves * 32, lds, part, s);
}

template <int CT>
hipError_t launch_f32_width(const RowsArgs &a, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    return w <= 64 ? launch_f32_full<CT, 64>(a, s) : w <= 128 ? launch_f32_full<CT, 128>(a, s) : launch_f32_full<CT, 256>(a, s);
}

}  // namespace

hipError_t launch_attend_rows_f32(const RowsArgs &a, hipStream_t s) {
    switch (a.c.type) {
        case 0: return launch_f32_width<0>(a, s);
        case 1: return launch_f32_width<1>(a, s);
        case 2: return launch_f32_width<2>(a, s);
        case 3: return launch_f32_width<3>(a, s);
        default: return launch_f32_width<4>(a, s);
    }
}

}  // namespace cqhip
