// gfx950 cross-attention of many query rows (nd_cross_attend_dev): 16-bit
// memories (cross_attend_kernel), and float32 ones (cross_attend_f32_kernel).
//
// Per (stream, key head) the query columns are the group's heads times the
// query rows, a wavefront holding 32 or 64 of them. Keys and values pass
// through LDS in tiles of 64 keys, two buffers, loaded straight into LDS
// (16 bytes a lane) one tile ahead and shared by the workgroup's four
// wavefronts. Both products run on the 32x32x16 matrix instruction with the
// columns last, so a lane keeps one column's maximum, sum and outputs:
//   S = K Q^T: A is 32 keys by 16 coordinates from LDS, B the query in
//     registers; lane (column n, half f) gets keys 8 (i / 4) + 4 f + i % 4 in
//     register i.
//   O = V^T P: a step contracts 16 keys in the order in which the lanes hold
//     them: the half f's eight are 4 f + {0..3} and 8 + 4 f + {0..3}, so the
//     weights are S's registers rounded in place and A's two halves are
//     transposing LDS reads (four keys by sixteen values each).
// The second product takes a weight in two parts of the memories' type, their
// sum off by 2^-16 of it in bfloat16 (a truncation, then the nearest to what
// that leaves) and 2^-22 in float16 (the nearest, twice). One part is off by
// 2^-9 and 2^-12, and the outputs' error against 64 bits was then 1.4 times
// that of their own rounding. The second costs its products, half as many
// again, and three vector operations a weight: 64 x 448 rows to 1500 frames,
// 8 heads of 64, 118 -> 156 us; 32 x 448 of 128 119 -> 145; 2 x 448 of 64
// 20.0 -> 21.7; 5 rows to 375 frames 9.0 -> 10.5. Logits, weights, their sums
// and the outputs are float32. The running maximum m is raised only when a
// column's logits pass it by 2^8, so most tiles leave the outputs unscaled.
// float16 weights are 2^(logit - m + 7): up to 2^15, which it holds, and none
// loses more than 2^-32 of the largest.
//
// Bank conflicts: row r of a tile keeps its 16-byte pieces in the order c ^
// f(r): f chosen so that sixteen lanes reading one piece of sixteen key rows,
// and the eight rows of four pieces of a transposing read, each cover all
// banks evenly.
#include "cq_internal.hpp"
#include "cq_device.hpp"
#include "tile_device.hpp"

#include <algorithm>
#include <type_traits>

namespace cqhip {
namespace {

constexpr int kXWaves = 4;
constexpr int kXTile = 64;

// The stream with the place-th longest memory (up to 64 streams). A launch of
// several rounds of workgroups takes the long ones first, so that none
// begins as the last ones end (40 ragged streams, 16 heads of 128 over 4: 109 ->
// 103 us).
__device__ __forceinline__ int longest_first(const SplitArgs &a, int place, int lane) {
    int n = -1;
    if (lane < a.batch) {
        const int mem = a.index ? a.index[lane] : lane;
        n = mem >= 0 && mem < a.memories ? min(max(a.k_len[mem], 0), a.nk_max) : 0;
    }
    int rank = 0;
    for (int j = 0; j < a.batch; ++j) {
        const int other = __builtin_amdgcn_readlane(n, j);
        rank += other > n || (other == n && j < lane);
    }
    return __ffsll(__ballot(lane < a.batch && rank == place)) - 1;
}

// D: widths up to D; CB: 32-column blocks a wavefront; FULL: both widths are
// D (else steps past a width are skipped by branches, which keep the
// compiler from interleaving the products with the softmax).
// The exponents s scale - m are rounded once (fmaf), so the largest is off 0 by
// the rounding of m = max(s) scale, at most half an ulp: the same factor in
// every weight of a column and their sum, and below 2^(1/32) as long as |m| is
// below 2^20. From there on, where it could leave float16 (from 2^28) or
// float32 (2^31), s scale is rounded first, as m is.
constexpr float kFar = 0x1p20f;
constexpr float kDown = 0x1p-8f;  // one over the largest weight, where the maximum lags
constexpr int kXFlags = 4 * kXWaves;  // bytes behind the tiles: an int a wavefront
template <int TYPE, int D, int CB, bool FULL>
__global__ __launch_bounds__(64 * kXWaves, D == 256 ? 1 : 2) void cross_attend_kernel(SplitArgs a, int col_tiles, int aligned) {
    constexpr int kPieces = D / 8;              // 16-byte pieces of a row
    constexpr int kLoads = D / 32;              // wavefront loads of a tile's keys (values) a wavefront
    constexpr int kLoadRows = 512 / D;          // rows of a wavefront load
    constexpr int kBytes = kXTile * D * 2;      // a tile's keys (values)
    extern __shared__ __align__(16) unsigned char smem[];  // [2][keys, values], flags

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    const XcdPlace x = xcd_place(a.batch * a.c.kv_heads, col_tiles * a.splits);  // a (stream, key head) on one XCD
    if (!x.ok) return;
    const int ct = x.within / a.splits, sp = x.within - ct * a.splits;
    int b = x.unit / a.c.kv_heads;
    const int h = x.unit - b * a.c.kv_heads;
    if (a.by_length) b = longest_first(a, b, lane);
    const int group = a.heads / a.c.kv_heads;
    const int mem = a.index ? a.index[b] : b;
    if (mem < 0 || mem >= a.memories) return;
    const int nk = a.k_len ? min(max(a.k_len[mem], 0), a.nk_max) : a.nk_max;
    const int cols = (a.q_len ? min(max(a.q_len[b], 0), a.t) : a.t) * group;
    constexpr int kWgCols = kXWaves * 32 * CB;
    if (ct * kWgCols >= cols) return;
    const int col0 = ct * kWgCols + wave * 32 * CB;
    const bool live = col0 < cols;
    const int per = ((nk + kXTile - 1) / kXTile + a.splits - 1) / a.splits * kXTile;
    const int j0 = min(sp * per, nk), j1 = min(j0 + per, nk);

    // The tiles' loads: piece c ^ f(row) of a row into place c.
    const unsigned char *kp = a.c.k + static_cast<long long>(mem) * a.k_mem + static_cast<long long>(h) * a.k_head;
    const unsigned char *vp = a.c.v + static_cast<long long>(mem) * a.v_mem + static_cast<long long>(h) * a.v_head;
    const int lrow = wave * kLoads * kLoadRows + lane / kPieces, lc = lane % kPieces;
    auto load_tile = [&](int j, int buf) {
        lds_bytes *base = (lds_bytes *)smem + buf * 2 * kBytes + wave * kLoads * 1024;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int row = lrow + k * kLoadRows, src = min(j + row, nk - 1);
            const int ck = (lc ^ k_swizzle<D>(row)) * 16, cv = (lc ^ v_swizzle<D>(row)) * 16;
            if (FULL || ck < 2 * a.c.qk)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(kp + src * a.k_row + ck),
                    (__attribute__((address_space(3))) void *)(base + k * 1024), 16, 0, 0);
            if (FULL || cv < 2 * a.c.vd)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(vp + src * a.v_row + cv),
                    (__attribute__((address_space(3))) void *)(base + kBytes + k * 1024), 16, 0, 0);
        }
    };
    // Values behind the last key: 0, not the last row's, whose infinities times
    // a weight of 0 are none. A wavefront clears what it loaded.
    auto clear_tail = [&](int j, int buf) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (j + lrow + k * kLoadRows >= j1)
                *reinterpret_cast<uint4 *>(smem + buf * 2 * kBytes + kBytes + (wave * kLoads + k) * 1024 + lane * 16) =
                    make_uint4(0, 0, 0, 0);
    };
    if (!FULL) {  // pieces past a row's width stay zero
        for (int x = tid * 16; x < 4 * kBytes; x += 64 * kXWaves * 16)
            *reinterpret_cast<uint4 *>(smem + x) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    // The queries: lane (n, half) holds coordinates 16 s + 8 half + 0..7 of its columns.
    s16x8 q[CB][D / 16];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int col = min(col0 + 32 * cb + n, cols - 1);
        const uint16_t *qp = static_cast<const uint16_t *>(a.q) + static_cast<long long>(b) * a.q_stream +
                             static_cast<long long>(col / group) * a.q_row +
                             static_cast<long long>(h * group + col % group) * a.c.qk;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const int d = 16 * s + 8 * half;
            s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
            if (FULL || 16 * s < a.c.qk) {
                if (aligned & 1) {
                    x = *reinterpret_cast<const s16x8 *>(qp + d);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = static_cast<short>(qp[d + e]);
                }
            }
            q[cb][s] = x;
        }
    }

    f32x16 o[CB][D / 32];
    float m[CB], l[CB];
    // LDS addresses: the keys' row n of a block, the values' row (lane % 16) / 4 and piece of a transposing read.
    const int kaddr = n * D * 2, kswz = k_swizzle<D>(n);
    const int ti = lane & 15, trow = 4 * half + (ti >> 2);
    const int vaddr = trow * D * 2 + 8 * (ti & 1), vpiece = 2 * ((lane >> 4) & 1) + ((ti & 3) >> 1), vswz = v_swizzle<D>(trow);

    // finite: the second parts, which may be 0 or below it, meet no infinite value,
    // and weights of bfloat16 memories are up to 1: 2^-8 of what they were, exactly.
    auto attend = [&](auto finite_values) {
        constexpr bool finite = decltype(finite_values)::value, down = finite && TYPE == 2;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            m[cb] = -INFINITY;
            l[cb] = 0.0f;
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[cb][v][i] = 0.0f;
        }
        if (j0 < j1) load_tile(j0, 0);
        int buf = 0;
        for (int j = j0; j < j1; j += kXTile, buf ^= 1) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (j + kXTile > j1) clear_tail(j, buf);
            __syncthreads();  // this tile is whole, and the other buffer's readers are done
            if (j + kXTile < j1) load_tile(j + kXTile, buf ^ 1);
            if (!live) continue;
            const unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
            f32x16 s[CB][2];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[cb][kb][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
                if (FULL || 16 * ks < a.c.qk) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const s16x8 ka = *reinterpret_cast<const s16x8 *>(kt + kb * 32 * D * 2 + kaddr + ((2 * ks + half) ^ kswz) * 16);
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb) s[cb][kb] = mfma16<TYPE>(ka, q[cb][ks], s[cb][kb]);
                    }
                }
            if (j + kXTile > j1) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (j + 32 * kb + 8 * (i >> 2) + 4 * half + (i & 3) >= j1) {
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb) s[cb][kb][i] = -INFINITY;
                        }
            }
            u32x4 p[CB][4], rest[CB][4];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                float mt = s[cb][0][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[cb][0][i]);
#pragma unroll
                for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[cb][1][i]);
                mt = halves_max(mt) * a.scale_log2;
                float scale = a.scale_log2;
                if (__any(mt > m[cb] + 8.0f || fabsf(m[cb]) >= kFar)) {
                    const float mn = fmaxf(m[cb], mt);
                    const float f = m[cb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[cb] - mn);
                    m[cb] = mn;
                    l[cb] *= f;
#pragma unroll
                    for (int v = 0; v < D / 32; ++v)
                        if (FULL || 32 * v < a.c.vd) o[cb][v] *= f;
                    const bool far = fabsf(mn) >= kFar;
                    if (__any(far)) {
                        const float first = far ? scale : 1.0f;
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[cb][0][i] *= first, s[cb][1][i] *= first;
                        scale = far ? 1.0f : scale;
                    }
                }
                const float mu = m[cb] == -INFINITY ? 0.0f : m[cb] - kLift<TYPE>;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float x = __builtin_amdgcn_exp2f(fmaf(s[cb][kb][i], scale, -mu));
                        float y = __builtin_amdgcn_exp2f(fmaf(s[cb][kb][i + 1], scale, -mu));
                        if constexpr (down) {
                            x *= kDown;
                            y *= kDown;
                        }
                        l[cb] += x;
                        l[cb] += y;
                        const uint32_t parts = first_parts<TYPE>(x, y);
                        p[cb][2 * kb + (i >> 3)][(i & 7) >> 1] = parts;
                        rest[cb][2 * kb + (i >> 3)][(i & 7) >> 1] = second_parts<TYPE>(x, y, parts);
                    }
            }
            // all first parts of 16 keys, then all second ones: no product waits for the one before it
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                s16x8 va[D / 32];
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    if (FULL || 32 * v < a.c.vd) {
                        const unsigned char *at = vt + 16 * st * D * 2 + vaddr + ((4 * v + vpiece) ^ vswz) * 16;
                        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
                        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4 *)(at + 8 * D * 2));
                        va[v] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb)
                            o[cb][v] = mfma16<TYPE>(va[v], __builtin_bit_cast(s16x8, p[cb][st]), o[cb][v]);
                    }
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    if (FULL || 32 * v < a.c.vd) {
                        if (finite) va[v] = finite16<TYPE>(va[v]);
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb)
                            o[cb][v] = mfma16<TYPE>(va[v], __builtin_bit_cast(s16x8, rest[cb][st]), o[cb][v]);
                    }
            }
        }
    };
    attend(std::false_type{});
    // A NaN: an infinite value may be behind it, which the first parts alone
    // make infinite; or a sum past kMostSum, of weights of up to 2^8.
    // All over again for the workgroup, whose wavefronts share the tiles.
    bool again = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int v = 0; v < D / 32; ++v)
#pragma unroll
            for (int i = 0; i < 16; ++i) again |= !(fabsf(o[cb][v][i]) < kMostSum);
    const bool wave_again = live && __any(again);
    int *flags = reinterpret_cast<int *>(smem + 4 * kBytes);
    if (lane == 0) flags[wave] = wave_again;
    __syncthreads();  // also: the tiles' readers are done
    const int4 any = *reinterpret_cast<const int4 *>(flags);
    const bool twice = any.x | any.y | any.z | any.w;
    if (twice) attend(std::true_type{});
    if (!live) return;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const float sum = halves_sum(l[cb]);
        const int col = col0 + 32 * cb + n;
        if (col >= cols) continue;
        const int head = h * group + col % group, row = col / group;
        if (a.part) {
            const long long pi = ((static_cast<long long>(b) * a.t + row) * a.heads + head) * a.splits + sp;
            float *dst = a.part + pi * a.c.vd;
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * v + 8 * g + 4 * half;
                    if (FULL || d < a.c.vd)
                        *reinterpret_cast<float4 *>(dst + d) =
                            make_float4(o[cb][v][4 * g], o[cb][v][4 * g + 1], o[cb][v][4 * g + 2], o[cb][v][4 * g + 3]);
                }
            if (half == 0) {
                a.part_ml[2 * pi] = m[cb] - (TYPE == 2 && twice ? -8.0f : kLift<TYPE>);
                a.part_ml[2 * pi + 1] = sum;
            }
        } else {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint16_t *dst = static_cast<uint16_t *>(a.out) + static_cast<long long>(b) * a.out_stream +
                            static_cast<long long>(row) * a.out_row + static_cast<long long>(head) * a.c.vd;
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * v + 8 * g + 4 * half;
                    if (FULL || d < a.c.vd) {
                        s16x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = round16<TYPE>(o[cb][v][4 * g + e] * inv);
                        if (aligned & 2) {
                            *reinterpret_cast<s16x4 *>(dst + d) = x;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) dst[d + e] = static_cast<uint16_t>(x[e]);
                        }
                    }
                }
        }
    }
}

// The same in float32, for many rows: 32 columns a wavefront on
// v_mfma_f32_32x32x2_f32. S = K q^T contracts a 16-byte piece of each half's
// coordinates in four instructions (element e of the halves' pieces in the
// e-th); O = V^T P takes S's register i as it lies (the half f's key is 8 (i /
// 4) + 4 f + i % 4) against one value of that key a lane. Tiles of 64 keys (32
// past heads of 64) through LDS as above; the weights stay float32, and meet the
// values as 2^-8 of what they are, so that sums of large values stay in range (of those
// under 1e-36 the subnormals' last bits are lost: 1e-5 of values of 1e-38). The value
// reads of the two halves, four rows apart, meet in no bank: rows with bit 2
// set keep their 128-byte halves exchanged.
template <int D, bool FULL>
__global__ __launch_bounds__(64 * kXWaves, D == 256 ? 1 : 2) void cross_attend_f32_kernel(SplitArgs a, int col_tiles) {
    constexpr int kKeys = D == 64 ? 64 : 32;   // keys a tile
    constexpr int kPieces = D / 4;             // 16-byte pieces of a row
    constexpr int kLoads = kKeys * D / 1024;   // wavefront loads of a tile's keys (values) a wavefront
    constexpr int kLoadRows = 256 / D;         // rows of a wavefront load
    constexpr int kBytes = kKeys * D * 4;
    extern __shared__ __align__(16) unsigned char smem[];  // [2][keys, values]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    const XcdPlace x = xcd_place(a.batch * a.c.kv_heads, col_tiles * a.splits);
    if (!x.ok) return;
    const int ct = x.within / a.splits, sp = x.within - ct * a.splits;
    int b = x.unit / a.c.kv_heads;
    const int h = x.unit - b * a.c.kv_heads;
    if (a.by_length) b = longest_first(a, b, lane);
    const int group = a.group;
    const int mem = a.index ? a.index[b] : b;
    if (mem < 0 || mem >= a.memories) return;
    const int nk = a.k_len ? min(max(a.k_len[mem], 0), a.nk_max) : a.nk_max;
    const int cols = (a.q_len ? min(max(a.q_len[b], 0), a.t) : a.t) * group;
    constexpr int kWgCols = kXWaves * 32;
    if (ct * kWgCols >= cols) return;
    const int col0 = ct * kWgCols + wave * 32;
    const bool live = col0 < cols;
    const int per = ((nk + kKeys - 1) / kKeys + a.splits - 1) / a.splits * kKeys;
    const int j0 = min(sp * per, nk), j1 = min(j0 + per, nk);

    const unsigned char *kp = a.c.k + static_cast<long long>(mem) * a.k_mem + static_cast<long long>(h) * a.k_head;
    const unsigned char *vp = a.c.v + static_cast<long long>(mem) * a.v_mem + static_cast<long long>(h) * a.v_head;
    const int lrow = wave * kLoads * kLoadRows + lane / kPieces, lc = lane % kPieces;
    auto load_tile = [&](int j, int buf) {
        lds_bytes *base = (lds_bytes *)smem + buf * 2 * kBytes + wave * kLoads * 1024;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int row = lrow + k * kLoadRows, src = min(j + row, nk - 1);
            const int ck = (lc ^ (row & 15)) * 16, cv = (lc ^ (((row >> 2) & 1) << 3)) * 16;
            if (FULL || ck < 4 * a.c.qk)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(kp + src * a.k_row + ck),
                    (__attribute__((address_space(3))) void *)(base + k * 1024), 16, 0, 0);
            if (FULL || cv < 4 * a.c.vd)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(vp + src * a.v_row + cv),
                    (__attribute__((address_space(3))) void *)(base + kBytes + k * 1024), 16, 0, 0);
        }
    };
    // Values behind the last key: 0, not the last row's, whose infinities times
    // a weight of 0 are none. A wavefront clears what it loaded.
    auto clear_tail = [&](int j, int buf) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (j + lrow + k * kLoadRows >= j1)
                *reinterpret_cast<uint4 *>(smem + buf * 2 * kBytes + kBytes + (wave * kLoads + k) * 1024 + lane * 16) =
                    make_uint4(0, 0, 0, 0);
    };
    if (!FULL) {  // pieces past a row's width stay zero
        for (int y = tid * 16; y < 4 * kBytes; y += 64 * kXWaves * 16)
            *reinterpret_cast<uint4 *>(smem + y) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    if (j0 < j1) load_tile(j0, 0);

    // The queries: lane (n, half) holds coordinates 8 s + 4 half + 0..3 of its column.
    float q[D / 2];
    {
        const int col = min(col0 + n, cols - 1);
        const float *qp = static_cast<const float *>(a.q) + static_cast<long long>(b) * a.q_stream +
                          static_cast<long long>(col / group) * a.q_row +
                          static_cast<long long>(h * group + col % group) * a.c.qk;
#pragma unroll
        for (int s = 0; s < D / 8; ++s) {
            const int d = 8 * s + 4 * half;
            float4 y = make_float4(0, 0, 0, 0);
            if (FULL || d < a.c.qk) {
                if (a.q_vec)
                    y = *reinterpret_cast<const float4 *>(qp + d);
                else
                    y = make_float4(qp[d], qp[d + 1], qp[d + 2], qp[d + 3]);
            }
            q[4 * s] = y.x * a.scale_log2;
            q[4 * s + 1] = y.y * a.scale_log2;
            q[4 * s + 2] = y.z * a.scale_log2;
            q[4 * s + 3] = y.w * a.scale_log2;
        }
    }
    f32x16 o[D / 32];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[v][i] = 0.0f;

    int buf = 0;
    for (int j = j0; j < j1; j += kKeys, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (j + kKeys > j1) clear_tail(j, buf);
        __syncthreads();  // this tile is whole, and the other buffer's readers are done
        if (j + kKeys < j1) load_tile(j + kKeys, buf ^ 1);
        if (!live) continue;
        const unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
#pragma unroll
        for (int kb = 0; kb < kKeys / 32; ++kb) {
            if (j + 32 * kb >= j1) break;
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
            const unsigned char *kr = kt + (32 * kb + n) * D * 4;
#pragma unroll
            for (int p = 0; p < D / 8; ++p)
                if (FULL || 8 * p < a.c.qk) {
                    const float4 ka = *reinterpret_cast<const float4 *>(kr + ((2 * p + half) ^ (n & 15)) * 16);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.x, q[4 * p], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.y, q[4 * p + 1], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.z, q[4 * p + 2], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(ka.w, q[4 * p + 3], s, 0, 0, 0);
                }
            if (j + 32 * kb + 32 > j1) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (j + 32 * kb + 8 * (i >> 2) + 4 * half + (i & 3) >= j1) s[i] = -INFINITY;
            }
            float mt = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
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
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i] - mu);
                l += s[i];
                s[i] *= kDown;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 32 * kb + 8 * (i >> 2) + 4 * half + (i & 3);
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    if (FULL || 32 * v < a.c.vd) {
                        const float va = *reinterpret_cast<const float *>(vt + row * D * 4 + (((32 * v + n) * 4) ^ (half << 7)));
                        o[v] = __builtin_amdgcn_mfma_f32_32x32x2f32(va, s[i], o[v], 0, 0, 0);
                    }
            }
        }
    }
    if (!live) return;
    const float sum = halves_sum(l);
    const int col = col0 + n;
    if (col >= cols) return;
    const int head = h * group + col % group, row = col / group;
    const long long pi = ((static_cast<long long>(b) * a.t + row) * a.heads + head) * a.splits + sp;
    float *dst = a.part ? a.part + pi * a.c.vd
                        : static_cast<float *>(a.out) + static_cast<long long>(b) * a.out_stream +
                              static_cast<long long>(row) * a.out_row + static_cast<long long>(head) * a.c.vd;
    const float f = a.part ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / (sum * kDown);
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * v + 8 * g + 4 * half;
            if (FULL || d < a.c.vd) {
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[d + e] = o[v][4 * g + e] * f;
            }
        }
    if (a.part && half == 0) {
        a.part_ml[2 * pi] = m;
        a.part_ml[2 * pi + 1] = sum * kDown;
    }
}

template <int TYPE, int D, int CB, bool FULL>
hipError_t launch_cross_full(const SplitArgs &a, int cols, int aligned, hipStream_t s) {
    constexpr int lds = 2 * 2 * kXTile * D * 2 + kXFlags;
    static std::atomic<unsigned long long> attr{0};
    if (lds > 64 * 1024)
        if (hipError_t e = lds_limit_once(reinterpret_cast<const void *>(&cross_attend_kernel<TYPE, D, CB, FULL>), lds, attr)) return e;
    const int col_tiles = (cols + kXWaves * 32 * CB - 1) / (kXWaves * 32 * CB);
    const long long grid = xcd_grid(static_cast<long long>(a.batch) * a.c.kv_heads, static_cast<long long>(col_tiles) * a.splits);
    hipLaunchKernelGGL((cross_attend_kernel<TYPE, D, CB, FULL>), dim3(static_cast<unsigned>(grid)), dim3(64 * kXWaves), lds, s,
                       a, col_tiles, aligned);
    return hipGetLastError();
}

template <int TYPE, int D, int CB>
hipError_t launch_cross(const SplitArgs &a, int cols, int aligned, hipStream_t s) {
    return a.c.qk == D && a.c.vd == D ? launch_cross_full<TYPE, D, CB, true>(a, cols, aligned, s)
                                      : launch_cross_full<TYPE, D, CB, false>(a, cols, aligned, s);
}

template <int TYPE>
hipError_t launch_cross_type(const SplitArgs &a, int cols, int cb, int aligned, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return cb == 2 ? launch_cross<TYPE, 64, 2>(a, cols, aligned, s) : launch_cross<TYPE, 64, 1>(a, cols, aligned, s);
    if (w <= 128) return launch_cross<TYPE, 128, 1>(a, cols, aligned, s);
    return launch_cross<TYPE, 256, 1>(a, cols, aligned, s);
}

// 64 columns a wavefront for heads of up to 64 once they still give every CU
// a workgroup: half the LDS reads an operation (448 rows to 1500 frames, 8
// heads of 64: 64 streams 156 us against 162 with 32 columns, 32 streams 80
// against 86, 16, just a workgroup a CU, 49 against 47; 2 streams, 32 workgroups
// of 64 columns a wavefront or 64 of 32: 25.5 against 21.7). Heads of 128 keep
// 32: 64 columns take the registers of a second wavefront a SIMD.
int column_blocks(const SplitArgs &a, int cus) {
    const long long cols = static_cast<long long>(a.t) * (a.heads / a.c.kv_heads), wide = kXWaves * 64;
    return a.type != 0 && std::max(a.c.qk, a.c.vd) <= 64 && (cols + wide - 1) / wide * a.batch * a.c.kv_heads >= cus ? 2 : 1;
}

template <int D, bool FULL>
hipError_t launch_cross_f32_full(const SplitArgs &a, int cols, hipStream_t s) {
    constexpr int lds = 2 * 2 * (D == 64 ? 64 : 32) * D * 4;
    static std::atomic<unsigned long long> attr{0};
    if (lds > 64 * 1024)
        if (hipError_t e = lds_limit_once(reinterpret_cast<const void *>(&cross_attend_f32_kernel<D, FULL>), lds, attr)) return e;
    const int col_tiles = (cols + kXWaves * 32 - 1) / (kXWaves * 32);
    const long long grid = xcd_grid(static_cast<long long>(a.batch) * a.c.kv_heads, static_cast<long long>(col_tiles) * a.splits);
    hipLaunchKernelGGL((cross_attend_f32_kernel<D, FULL>), dim3(static_cast<unsigned>(grid)), dim3(64 * kXWaves), lds, s, a,
                       col_tiles);
    return hipGetLastError();
}

template <int D>
hipError_t launch_cross_f32(const SplitArgs &a, int cols, hipStream_t s) {
    return a.c.qk == D && a.c.vd == D ? launch_cross_f32_full<D, true>(a, cols, s) : launch_cross_f32_full<D, false>(a, cols, s);
}

}  // namespace

int cross_workgroup_columns(const SplitArgs &a, int cus) { return kXWaves * 32 * column_blocks(a, cus); }

hipError_t launch_cross_attend(const SplitArgs &args, int cus, hipStream_t s) {
    SplitArgs a = args;
    const int cols = a.t * (a.heads / a.c.kv_heads), cb = column_blocks(a, cus);
    const long long tiles = (cols + kXWaves * 32 * cb - 1) / (kXWaves * 32 * cb);
    a.by_length = a.k_len && a.batch <= 64 && tiles * a.batch * a.c.kv_heads > 2LL * cus;
    // queries readable in 16-byte pieces, outputs writable in 8-byte ones
    int aligned = 0;
    if (((reinterpret_cast<uintptr_t>(a.q) | (a.q_stream * 2) | (a.q_row * 2)) & 15) == 0) aligned |= 1;
    if (((reinterpret_cast<uintptr_t>(a.out) | (a.out_stream * 2) | (a.out_row * 2)) & 7) == 0) aligned |= 2;
    hipError_t e;
    const int w = std::max(a.c.qk, a.c.vd);
    if (a.type == 0)
        e = w <= 64 ? launch_cross_f32<64>(a, cols, s) : w <= 128 ? launch_cross_f32<128>(a, cols, s) : launch_cross_f32<256>(a, cols, s);
    else
        e = a.type == 1 ? launch_cross_type<1>(a, cols, cb, aligned, s) : launch_cross_type<2>(a, cols, cb, aligned, s);
    if (e != hipSuccess || !a.part) return e;
    return launch_attend_join(a, s);
}

}  // namespace cqhip
