// gfx950 causal attention of many rows over paged float32 caches
// (rows_kernels.hip describes the tiles, the masks and the columns computed again).
//
// What bounds it: 16 prompts of 448 rows, 8 heads of 64, 64 to 73 us (21.5 at the rate
// of a large float32 product): one round of workgroups, of which the first rows' walk 128
// keys and the last rows' all; matrix units busy 34% of all cycles, CUs 71%. 8 prompts of 2000
// rows 355 us (214), 63% and 86%. Heads past 128 leave one workgroup a CU, whose four
// wavefronts wait half of their cycles: 16 prompts, 8 heads of 240 over 4, 300 to 370 us (81).
#include "rows_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

// 32 columns a wavefront on v_mfma_f32_32x32x2_f32, the products of
// cross_attend_f32_kernel. FULL: both widths are D. Else the tiles and queries are 0
// past a width, and with SKIP no products are made there: branches that keep the
// compiler from interleaving, taken where they leave out a quarter of wide heads or
// more (16 prompts of 448 rows, 8 heads over 4 of 144: 278 us, 355 without; of 240: 460
// and 370; of 80 116 and 111; 8 heads of 16 79 and 71, of 48 162 and 74).
template <int D, bool FULL, bool SKIP>
__global__ __launch_bounds__(64 * kRWaves, D == 256 ? 1 : 2) void rows_attend_f32_kernel(RowsArgs a, int col_tiles) {
    constexpr int kKeys = D == 64 ? 64 : 32;   // keys a tile
    constexpr int kBytes = kKeys * D * 4;
    constexpr int kRowPieces = D / 4;             // 16-byte pieces of a row
    constexpr int kStage = kKeys * kRowPieces / 256;  // pieces a thread stages
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
    float4 kst[kStage], vst[kStage];
    auto fetch = [&](int rows) {
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kRowPieces, c = piece % kRowPieces;
            const long long src = __shfl(rows, row);
            kst[k] = FULL || 4 * c < a.c.qk ? *reinterpret_cast<const float4 *>(kp + src * a.k_row + c * 16) : make_float4(0, 0, 0, 0);
            vst[k] = FULL || 4 * c < a.c.vd ? *reinterpret_cast<const float4 *>(vp + src * a.v_row + c * 16) : make_float4(0, 0, 0, 0);
        }
    };
    auto store = [&](int j, int buf) {
        unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kRowPieces, c = piece % kRowPieces;
            *reinterpret_cast<float4 *>(kt + row * D * 4 + ((c ^ (row & 15)) * 16)) = kst[k];
            // values behind the last key: 0
            *reinterpret_cast<float4 *>(vt + row * D * 4 + ((c ^ (((row >> 2) & 1) << 3)) * 16)) =
                j + row >= p.end ? make_float4(0, 0, 0, 0) : vst[k];
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
            for (int c = 0; c < D / 8; ++c) {
                if (SKIP && 8 * c >= a.c.qk) break;
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
                for (int v = 0; v < D / 32; ++v) {
                    if (SKIP && 32 * v >= a.c.vd) break;
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
    bool again = false;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) again |= !(fabsf(o[v][e]) < kMostSum);
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
    const unsigned long long bad = __ballot(again && col < p.cols);
    if (bad) repair_columns<kKeys>(a, p, col0, static_cast<unsigned>(bad) | static_cast<unsigned>(bad >> 32));
}

template <int D>
hipError_t launch_f32(const RowsArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> full{0}, part{0}, skip{0};
    constexpr int lds = 4 * (D == 64 ? 64 : 32) * D * 4;
    if (a.c.qk == D && a.c.vd == D) return launch_with(&rows_attend_f32_kernel<D, true, false>, a, kRWaves * 32, lds, full, s);
    if constexpr (D == 256)
        if (4 * std::max(a.c.qk, a.c.vd) <= 3 * D) return launch_with(&rows_attend_f32_kernel<D, false, true>, a, kRWaves * 32, lds, skip, s);
    return launch_with(&rows_attend_f32_kernel<D, false, false>, a, kRWaves * 32, lds, part, s);
}

}  // namespace

hipError_t launch_attend_rows_f32(const RowsArgs &a, hipStream_t s) {
    if (a.c.type != 0) return hipErrorInvalidValue;  // the split form has them
    const int w = std::max(a.c.qk, a.c.vd);
    return w <= 64 ? launch_f32<64>(a, s) : w <= 128 ? launch_f32<128>(a, s) : launch_f32<256>(a, s);
}

}  // namespace cqhip
