// gfx950 causal attention of many rows a stream over paged caches of any type,
// with a window and first rows that stay visible (kv_attend_rows_paged_dev).
//
// Per (stream, key head) the query columns are the rows times the group's
// heads, 32 a wavefront. Tiles of 64 keys (32 for wide float32 heads)
// pass through LDS, two buffers, shared by the workgroup's four wavefronts;
// both products run on 32x32 matrix instructions with the columns last, so a
// lane keeps one column's maximum, sum and outputs (the lane orders of
// cross_kernels.hip). A workgroup walks the tiles that any of its columns
// sees: the first `sink` keys', then those from its first row's window to its
// last row; a wavefront skips what none of its columns sees and compares
// positions only in tiles that some see in part.
//
// rows_attend_kernel, 16-bit queries over caches of their type or of 8 bits:
// 32x32x16 products. Caches of the queries' type go straight into LDS; codes
// pass through registers, widened exactly (keys to the queries' type, values to
// bfloat16, whose range holds a weight of 1 times any scale): a key's scale meets
// its logit, a value's scale its weight. Weights take part as the sum of two
// parts of the values' type (22 bits in float16, 16 in bfloat16).
// rows_attend_f32_kernel, queries of any type over float32 caches: 32x32x2
// products, all of it in float32. The other pairs of types take the split form
// (parts_kernels.hip) at any number of columns.
//
// What bounds 8 ragged prompts of up to 2000 rows, 16 heads of 128 over 4 in
// bfloat16 (220 to 226 us, some 600 TFLOP/s): the softmax on the vector units, 45% of all
// cycles, beside the products, 42%, with little overlap. 4 of up to 1000 rows over
// int8 pages with a window of 1024, 16 heads of 64 over 4: 47 to 54 us, half of the CUs' cycles idle. 8 whole
// prompts of 2000 rows over e4m3 pages, heads as the first: 233 to 264 us (bfloat16 caches 209), the
// vector units 49%, the products 36%.
//
// A masked key has the weight 0, but 0 times an infinite or NaN value is NaN,
// and so is a second part times an infinity: a wavefront that finds a NaN, or a
// sum that its parts' may bring past float32's range (kMostSum), among its
// outputs computes those columns again key by key (repair_columns), which skips
// masked keys. Keys behind the workgroup's last are cleared.
#include "rows_device.hpp"

#include <algorithm>
#include <cstring>

namespace cqhip {
namespace {

// Codes two at a time as two values of a 16-bit type (1 float16, 2 bfloat16), exactly.
template <int CODE, int TYPE>
__device__ __forceinline__ uint32_t widen2(uint32_t w, int pair) {
    float x, y;
    if constexpr (CODE == 3) {
        x = static_cast<float>(static_cast<int32_t>(w << (24 - 16 * pair)) >> 24);
        y = static_cast<float>(static_cast<int32_t>(w << (16 - 16 * pair)) >> 24);
    } else {
        const auto v = pair ? __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true)
                            : __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        x = v[0];
        y = v[1];
    }
    if constexpr (TYPE == 1) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
}

constexpr float kRowsFar = 0x1p20f;  // from a maximum of it on, logits are rounded before it is subtracted, as it was

// QT: the queries' type (1 float16, 2 bfloat16); CT: the cache's (QT itself, 3
// int8, 4 e4m3); D: widths up to D; FULL: both widths are D, else the tiles and
// queries are 0 past a width and take part like others (branches around
// those products keep the compiler from interleaving them with the softmax: 64 prompts
// of 448 rows, 8 heads of 48 over 2, 96 us against 44; 32 of 80, 58 and 44).
// 64 columns a wavefront, at half the LDS reads a product, lost too: 64 prompts of up to 448
// rows, 8 heads of 64, 48 us against 36; 8 of 2000 rows, 16 heads over 4, 144 and 136.
// KS: 1, or 2 where few columns would leave wavefronts or CUs idle: wavefronts 0 and
// 1 take the first 32 keys of a tile, 2 and 3 the others, joined at the end.
template <int QT, int CT, int D, int KS, bool FULL>
__global__ __launch_bounds__(64 * kRWaves, D == 256 ? 1 : 2) void rows_attend_kernel(RowsArgs a, int col_tiles) {
    constexpr bool kCodes = CT >= 3;
    constexpr int VT = kCodes ? 2 : QT;          // the values' type in LDS
    constexpr int kPieces = D / 8;               // 16-byte pieces of a row in LDS
    constexpr int kLoads = D / 32;               // wavefront loads of a tile's keys (values) a wavefront
    constexpr int kLoadRows = 512 / D;           // rows of a wavefront load
    constexpr int kBytes = kRTile * D * 2;       // a tile's keys (values)
    constexpr int kStage = kCodes ? D / 64 : 1;  // 16-byte pieces of codes a thread stages
    extern __shared__ __align__(16) unsigned char smem[];  // [2][keys, values], [2][key scales, value scales]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    constexpr int kWgCols = kRWaves / KS * 32;
    constexpr int kBlocks = 2 / KS;              // blocks of 32 keys of a tile a wavefront takes
    const RowsPlace p = rows_place<kRTile>(a, col_tiles, kWgCols);
    if (!p.ok) return;
    const int col_wave = wave % (kRWaves / KS), block0 = wave / (kRWaves / KS);
    const int col0 = p.ct * kWgCols + col_wave * 32;
    const bool live = col0 < p.cols;
    // the wavefront's rows' positions, its columns' own
    const int first = p.pos + min(col0, p.cols - 1) / a.group, last = p.pos + (min(col0 + 32, p.cols) - 1) / a.group;
    const int at = p.pos + min(col0 + n, p.cols - 1) / a.group;

    const unsigned char *kp = a.c.k + static_cast<long long>(p.h) * a.k_head;
    const unsigned char *vp = a.c.v + static_cast<long long>(p.h) * a.v_head;
    float *scales = reinterpret_cast<float *>(smem + 4 * kBytes);

    // The pool row of key `lane` of tile i; keys behind the last read that one's.
    auto rows_of = [&](int i) { return pool_row(a, p.b, min(tile_key<kRTile>(p, i) + lane, p.end - 1)); };
    // Caches of the queries' type: piece c ^ f(row) of a row into place c.
    const int lrow = wave * kLoads * kLoadRows + lane / kPieces, lc = lane % kPieces;
    auto load_tile = [&](int rows, int buf) {
        lds_bytes *base = (lds_bytes *)smem + buf * 2 * kBytes + wave * kLoads * 1024;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int row = lrow + k * kLoadRows;
            const long long src = __shfl(rows, row);
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
    // Values behind the last key: 0. A wavefront clears what it loaded.
    auto clear_tail = [&](int j, int buf) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (j + lrow + k * kLoadRows >= p.end)
                *reinterpret_cast<uint4 *>(smem + buf * 2 * kBytes + kBytes + (wave * kLoads + k) * 1024 + lane * 16) =
                    make_uint4(0, 0, 0, 0);
    };
    // Codes: 16 of a row a piece, thread tid the pieces tid + 256 k, through registers.
    constexpr int kCodePieces = D / 16;
    uint4 kst[kStage], vst[kStage];
    float sst = 0.0f;
    auto fetch_codes = [&](int rows) {
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kCodePieces, c = piece % kCodePieces * 16;
            const long long src = __shfl(rows, row & 63);
            kst[k] = FULL || c < a.c.qk ? *reinterpret_cast<const uint4 *>(kp + src * a.k_row + c) : make_uint4(0, 0, 0, 0);
            vst[k] = FULL || c < a.c.vd ? *reinterpret_cast<const uint4 *>(vp + src * a.v_row + c) : make_uint4(0, 0, 0, 0);
        }
        if (wave < 2) sst = (wave ? a.c.vs : a.c.ks)[static_cast<long long>(rows >> a.c.sshift) * a.c.kv_heads + p.h];
    };
    auto store_codes = [&](int j, int buf) {
        unsigned char *kt = smem + buf * 2 * kBytes, *vt = kt + kBytes;
#pragma unroll
        for (int k = 0; k < kStage; ++k) {
            const int piece = tid + 256 * k, row = piece / kCodePieces, c = piece % kCodePieces;
            const bool dead = j + row >= p.end;  // behind the last key: 0
            const uint32_t kw[4] = {kst[k].x, kst[k].y, kst[k].z, kst[k].w}, vw[4] = {vst[k].x, vst[k].y, vst[k].z, vst[k].w};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint4 x = make_uint4(widen2<CT, QT>(kw[2 * e], 0), widen2<CT, QT>(kw[2 * e], 1), widen2<CT, QT>(kw[2 * e + 1], 0),
                                     widen2<CT, QT>(kw[2 * e + 1], 1));
                *reinterpret_cast<uint4 *>(kt + row * D * 2 + ((2 * c + e) ^ k_swizzle<D>(row)) * 16) = x;
                x = make_uint4(widen2<CT, VT>(vw[2 * e], 0), widen2<CT, VT>(vw[2 * e], 1), widen2<CT, VT>(vw[2 * e + 1], 0),
                               widen2<CT, VT>(vw[2 * e + 1], 1));
                if (dead) x = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4 *>(vt + row * D * 2 + ((2 * c + e) ^ v_swizzle<D>(row)) * 16) = x;
            }
        }
        if (wave < 2) scales[(2 * buf + wave) * kRTile + lane] = j + lane >= p.end ? 0.0f : sst;
    };
    if (!FULL && !kCodes) {  // pieces past a row's width stay zero
        for (int x = tid * 16; x < 4 * kBytes; x += 64 * kRWaves * 16)
            *reinterpret_cast<uint4 *>(smem + x) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    // The queries: lane (n, half) holds coordinates 16 s + 8 half + 0..7 of its column.
    s16x8 q[D / 16];
    const int qcol = min(col0 + n, p.cols - 1);
    const uint16_t *qp = static_cast<const uint16_t *>(a.q) + static_cast<long long>(p.b) * a.q_stream +
                         static_cast<long long>(qcol / a.group) * a.q_row +
                         static_cast<long long>(p.h * a.group + qcol % a.group) * a.c.qk;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const int d = 16 * s + 8 * half;
        s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
        if (FULL || 16 * s < a.c.qk) {
            if (a.aligned & 1) {
                x = *reinterpret_cast<const s16x8 *>(qp + d);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = static_cast<short>(qp[d + e]);
            }
        }
        q[s] = x;
    }

    f32x16 o[D / 32];
    // LDS addresses: the keys' row n of a block, the values' row (lane % 16) / 4 and piece of a transposing read.
    const int kaddr = n * D * 2, kswz = k_swizzle<D>(n);
    const int ti = lane & 15, trow = 4 * half + (ti >> 2);
    const int vaddr = trow * D * 2 + 8 * (ti & 1), vpiece = 2 * ((lane >> 4) & 1) + ((ti & 3) >> 1), vswz = v_swizzle<D>(trow);
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[v][i] = 0.0f;

    // Rows are looked up two tiles ahead, tiles loaded one ahead.
    int rows = 0;
    if (p.i0 < p.i1) {
        rows = rows_of(p.i0);
        if constexpr (kCodes) {
            fetch_codes(rows);
            store_codes(tile_key<kRTile>(p, p.i0), 0);
        } else {
            load_tile(rows, 0);
        }
        if (p.i0 + 1 < p.i1) rows = rows_of(p.i0 + 1);
    }
    int buf = 0;
    for (int i = p.i0; i < p.i1; ++i, buf ^= 1) {
        const int j = tile_key<kRTile>(p, i);
        if constexpr (!kCodes) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (j + kRTile > p.end) clear_tail(j, buf);
        }
        __syncthreads();  // this tile is whole, and the other buffer's readers are done
        const bool more = i + 1 < p.i1;
        if (more) {
            if constexpr (kCodes)
                fetch_codes(rows);
            else
                load_tile(rows, buf ^ 1);
            if (i + 2 < p.i1) rows = rows_of(i + 2);
        }
        const int jw = j + 32 * block0;  // the wavefront's keys of the tile
        if (live && !none_sees(a, first, last, jw, jw + 32 * kBlocks - 1)) {
            const unsigned char *kt = smem + buf * 2 * kBytes + block0 * 32 * D * 2, *vt = kt + kBytes;
            f32x16 s[kBlocks];
#pragma unroll
            for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                for (int kb = 0; kb < kBlocks; ++kb) {
                    const s16x8 ka = *reinterpret_cast<const s16x8 *>(kt + kb * 32 * D * 2 + kaddr + ((2 * ks + half) ^ kswz) * 16);
                    s[kb] = mfma16<QT>(ka, q[ks], s[kb]);
                }
            if constexpr (kCodes) {
                const float *ks = scales + 2 * buf * kRTile + 32 * block0 + 4 * half;
#pragma unroll
                for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 x = *reinterpret_cast<const float4 *>(ks + 32 * kb + 8 * g);
                        s[kb][4 * g] *= x.x;
                        s[kb][4 * g + 1] *= x.y;
                        s[kb][4 * g + 2] *= x.z;
                        s[kb][4 * g + 3] *= x.w;
                    }
            }
            if (!all_see(a, first, last, jw, jw + 32 * kBlocks - 1)) {
#pragma unroll
                for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = jw + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3);
                        s[kb][e] = sees(a, at, key) ? s[kb][e] : -INFINITY;
                    }
            }
            u32x4 w[2 * kBlocks], rest[2 * kBlocks];
            float mt = s[0][0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mt = fmaxf(mt, s[0][e]);
            if constexpr (kBlocks == 2) {
#pragma unroll
                for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[1][e]);
            }
            mt = halves_max(mt) * a.scale_log2;
            float scale = a.scale_log2;
            if (__any(mt > m + 8.0f || fabsf(m) >= kRowsFar)) {
                const float mn = fmaxf(m, mt);
                const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int v = 0; v < D / 32; ++v) o[v] *= f;
                const bool far = fabsf(mn) >= kRowsFar;
                if (__any(far)) {
                    const float one = far ? scale : 1.0f;
#pragma unroll
                    for (int kb = 0; kb < kBlocks; ++kb) s[kb] *= one;
                    scale = far ? 1.0f : scale;
                }
            }
            const float mu = m == -INFINITY ? 0.0f : m - kLift<VT>;
            const float *vs = scales + (2 * buf + 1) * kRTile + 32 * block0 + 4 * half;
#pragma unroll
            for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    float x = __builtin_amdgcn_exp2f(fmaf(s[kb][e], scale, -mu));
                    float y = __builtin_amdgcn_exp2f(fmaf(s[kb][e + 1], scale, -mu));
                    l += x;
                    l += y;
                    if constexpr (kCodes) {
                        const float2 f = *reinterpret_cast<const float2 *>(vs + 32 * kb + 8 * (e >> 2) + (e & 3));
                        x *= f.x;
                        y *= f.y;
                    }
                    const uint32_t parts = first_parts<VT>(x, y);
                    w[2 * kb + (e >> 3)][(e & 7) >> 1] = parts;
                    rest[2 * kb + (e >> 3)][(e & 7) >> 1] = second_parts<VT>(x, y, parts);
                }
            // all first parts of 16 keys, then all second ones: no product waits for the one before it
#pragma unroll
            for (int st = 0; st < 2 * kBlocks; ++st) {
                s16x8 va[D / 32];
#pragma unroll
                for (int v = 0; v < D / 32; ++v) {
                    const unsigned char *src = vt + 16 * st * D * 2 + vaddr + ((4 * v + vpiece) ^ vswz) * 16;
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)src);
                    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4 *)(src + 8 * D * 2));
                    va[v] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[v] = mfma16<VT>(va[v], __builtin_bit_cast(s16x8, w[st]), o[v]);
                }
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    o[v] = mfma16<VT>(va[v], __builtin_bit_cast(s16x8, rest[st]), o[v]);
            }
        }
        if constexpr (kCodes)
            if (more) store_codes(tile_key<kRTile>(p, i + 1), buf ^ 1);
    }
    if constexpr (KS == 2) {
        // the other half's outputs, maximum and sum, from LDS: registers side by side
        constexpr int kRegs = D / 2 + 2;
        float *join = reinterpret_cast<float *>(smem) + col_wave * kRegs * 64 + lane;
        __syncthreads();  // the tiles' readers are done
        if (block0 == 1) {
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int e = 0; e < 16; ++e) join[(16 * v + e) * 64] = o[v][e];
            join[D / 2 * 64] = m;
            join[(D / 2 + 1) * 64] = l;
        }
        __syncthreads();
        if (block0 == 1) return;
        const float m1 = join[D / 2 * 64], mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - mu), f1 = __builtin_amdgcn_exp2f(m1 - mu);
        m = mn;
        l = l * f0 + join[(D / 2 + 1) * 64] * f1;
#pragma unroll
        for (int v = 0; v < D / 32; ++v)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[v][e] = o[v][e] * f0 + join[(16 * v + e) * 64] * f1;
    }
    if (!live) return;
    const int col = col0 + n;
    const float sum = halves_sum(l);
    bool again = false;
#pragma unroll
    for (int v = 0; v < D / 32; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) again |= !(fabsf(o[v][e]) < kMostSum);
    if (col < p.cols) {
        const int head = p.h * a.group + col % a.group, row = col / a.group;
        if (a.part) {
            const long long pi = ((static_cast<long long>(p.b) * a.t + row) * a.heads + head) * a.splits + p.sp;
            float *dst = a.part + pi * a.c.vd;
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * v + 8 * g + 4 * half;
                    if (FULL || d < a.c.vd)
                        *reinterpret_cast<float4 *>(dst + d) = make_float4(o[v][4 * g], o[v][4 * g + 1],
                                                                           o[v][4 * g + 2], o[v][4 * g + 3]);
                }
            if (half == 0) {
                a.part_ml[2 * pi] = m - kLift<VT>;
                a.part_ml[2 * pi + 1] = sum;
            }
        } else {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint16_t *dst = static_cast<uint16_t *>(a.out) + static_cast<long long>(p.b) * a.out_stream +
                            static_cast<long long>(row) * a.out_row + static_cast<long long>(head) * a.c.vd;
#pragma unroll
            for (int v = 0; v < D / 32; ++v)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * v + 8 * g + 4 * half;
                    if (FULL || d < a.c.vd) {
                        s16x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = round16<QT>(o[v][4 * g + e] * inv);
                        if (a.aligned & 2) {
                            *reinterpret_cast<s16x4 *>(dst + d) = x;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) dst[d + e] = static_cast<uint16_t>(x[e]);
                        }
                    }
                }
        }
    }
    const unsigned long long bad = __ballot(again && col < p.cols);
    if (bad) repair_columns<kRTile>(a, p, col0, static_cast<unsigned>(bad) | static_cast<unsigned>(bad >> 32));
}

template <int QT, int CT, int D, int KS, bool FULL>
hipError_t launch_16(const RowsArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> attr{0};
    constexpr int lds = 4 * kRTile * D * 2 + (CT >= 3 ? 4 * kRTile * 4 : 0);
    static_assert(KS == 1 || kRWaves / KS * (D / 2 + 2) * 64 * 4 <= lds, "the join's registers past the tiles");
    return launch_with(&rows_attend_kernel<QT, CT, D, KS, FULL>, a, kRWaves / KS * 32, lds, attr, s);
}

template <int QT, int CT, int D, int KS>
hipError_t launch_16_full(const RowsArgs &a, hipStream_t s) {
    return a.c.qk == D && a.c.vd == D ? launch_16<QT, CT, D, KS, true>(a, s) : launch_16<QT, CT, D, KS, false>(a, s);
}

template <int QT, int CT>
hipError_t launch_16_width(const RowsArgs &a, int ks, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return ks == 2 ? launch_16_full<QT, CT, 64, 2>(a, s) : launch_16_full<QT, CT, 64, 1>(a, s);
    if (w <= 128) return ks == 2 ? launch_16_full<QT, CT, 128, 2>(a, s) : launch_16_full<QT, CT, 128, 1>(a, s);
    return ks == 2 ? launch_16_full<QT, CT, 256, 2>(a, s) : launch_16_full<QT, CT, 256, 1>(a, s);
}

// 16-bit products: queries of 16 bits over a cache of their type or of codes.
bool rows_16(const RowsArgs &a) { return a.type != 0 && (a.c.type == a.type || a.c.type >= 3); }

// In how many parts a workgroup's wavefronts take a tile's keys: in halves where 64
// columns are all or workgroups of 128 do not give every CU two (a prompt of 448 rows,
// 8 heads of 64: 14.3 us whole, 11.0 in halves; 2 of 500 rows behind 2500 keys, 16
// heads of 128 over 4: 69 and 60; 4 of 1000, 512 such workgroups: 56 and 59).
int rows_key_parts(const RowsArgs &a, int cus) {
    if (!rows_16(a)) return 1;
    const long long cols = static_cast<long long>(a.t) * a.group;
    const long long blocks = (cols + kRWaves * 32 - 1) / (kRWaves * 32) * a.batch * a.c.kv_heads;
    return cols <= kRWaves / 2 * 32 || blocks < 2LL * cus ? 2 : 1;
}

}  // namespace

int rows_workgroup_columns(const RowsArgs &a, int cus) { return kRWaves / rows_key_parts(a, cus) * 32; }

hipError_t launch_attend_rows(const RowsArgs &args, int cus, hipStream_t s) {
    RowsArgs a = args;
    const int size = a.type == 0 ? 4 : 2;
    a.aligned = 0;
    if (((reinterpret_cast<uintptr_t>(a.q) | (a.q_stream * size) | (a.q_row * size)) & 15) == 0) a.aligned |= 1;
    if (((reinterpret_cast<uintptr_t>(a.out) | (a.out_stream * size) | (a.out_row * size)) & 7) == 0) a.aligned |= 2;
    hipError_t e;
    if (rows_16(a)) {
        const int ks = rows_key_parts(a, cus);
        if (a.type == 1)
            e = a.c.type == 1 ? launch_16_width<1, 1>(a, ks, s) : a.c.type == 4 ? launch_16_width<1, 4>(a, ks, s) : launch_16_width<1, 3>(a, ks, s);
        else
            e = a.c.type == 2 ? launch_16_width<2, 2>(a, ks, s) : a.c.type == 4 ? launch_16_width<2, 4>(a, ks, s) : launch_16_width<2, 3>(a, ks, s);
    } else {
        e = launch_attend_rows_f32(a, s);
    }
    if (e != hipSuccess || !a.part) return e;
    SplitArgs p;  // what the join reads
    std::memset(&p, 0, sizeof p);
    p.c = a.c;
    p.q_len = a.rows;
    p.pos = a.pos;
    p.nk_max = a.nk_max;
    p.t = a.t;
    p.heads = a.heads;
    p.batch = a.batch;
    p.splits = a.splits;
    p.out = a.out;
    p.out_stream = a.out_stream;
    p.out_row = a.out_row;
    p.type = a.type;
    p.part = a.part;
    p.part_ml = a.part_ml;
    return launch_attend_join(p, s);
}

}  // namespace cqhip
