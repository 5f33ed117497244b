// What the kernels of rows_kernels.hip and rows_f32_kernels.hip share: a
// workgroup's keys, the mask, the way through the pages, and the columns that
// are computed again.
#pragma once

#include "cq_internal.hpp"
#include "cq_device.hpp"
#include "tile_device.hpp"

namespace cqhip {

constexpr int kRWaves = 4;
constexpr int kRTile = 64;

// What a workgroup works on: its columns [col0, cols) of a stream's key head,
// and its keys as tiles of KEYS: `ns` from row 0 on, the others from lo on, in
// [i0, i1) of them, up to row end.
struct RowsPlace {
    int b, h, ct, sp, cols, pos, end, lo, ns, i0, i1;
    bool ok;
};
// Streams of unequal counts, of 1, 2, 4 or 8 key heads: a key head of all streams on
// 8 / kv_heads XCDs, whose L2s it shares with no other, its tiles of columns in turns, each turn of
// the streams one place on. Against lists spread over all XCDs, or whole ones
// on one where there are 64 or more (us a call): 8 prompts of up to 2000 rows, 16 heads of 128 over
// 4, 226 and 239; 6 of 1000, 8 heads of 64, 21 and 25; 64 of 448, 29 and 34; 32 of
// 448, 8 heads of 128 over 2, 27 and 32; without the turns 98 became 130. One head of 100
// equal streams, ten tiles each: 36 and 31.
__host__ __device__ inline bool rows_by_head(const RowsArgs &a) {
    return a.rows && 8 % a.c.kv_heads == 0 && (a.c.kv_heads > 1 || a.batch < kXcdUnits);
}
template <int KEYS>
__device__ __forceinline__ RowsPlace rows_place(const RowsArgs &a, int col_tiles, int wg_cols) {
    RowsPlace p;
    p.ok = false;
    // A (stream, key head) on one XCD; but streams of unequal counts by heads, or, where
    // there are few, over all of them: tile by tile, each turn of the units one place on.
    const int units = a.batch * a.c.kv_heads;
    XcdPlace x;
    if (rows_by_head(a)) {
        const int each = 8 / a.c.kv_heads, xcd = blockIdx.x & 7, slot = static_cast<int>(blockIdx.x) >> 3, turn = slot / a.batch;
        x.within = turn * each + xcd / a.c.kv_heads;
        x.unit = (slot - turn * a.batch + turn) % a.batch * a.c.kv_heads + xcd % a.c.kv_heads;
        if (x.within >= col_tiles * a.splits) return p;
    } else if (a.rows && units < kXcdUnits) {
        x.within = static_cast<int>(blockIdx.x) / units;
        x.unit = (static_cast<int>(blockIdx.x) - x.within * units + x.within) % units;
    } else {
        x = xcd_place(units, col_tiles * a.splits);
        if (!x.ok) return p;
    }
    const int ct = x.within / a.splits;
    p.sp = x.within - ct * a.splits;
    p.ct = col_tiles - 1 - ct;  // the last rows, which see most keys, first
    p.b = x.unit / a.c.kv_heads;
    p.h = x.unit - p.b * a.c.kv_heads;
    const int n = a.rows ? a.rows[p.b] : a.t;
    p.pos = a.pos[p.b];
    if (n <= 0 || n > a.t || p.pos < 0 || p.pos > a.nk_max - n) return p;
    p.cols = n * a.group;
    const int col0 = p.ct * wg_cols;
    if (col0 >= p.cols) return p;
    const int first = col0 / a.group, last = min(col0 + wg_cols, p.cols) - 1;
    p.end = p.pos + last / a.group + 1;
    p.lo = a.window ? max(p.pos + first - a.window + 1, 0) / KEYS * KEYS : 0;
    p.ns = a.window ? (min(a.sink, p.lo) + KEYS - 1) / KEYS : 0;
    if (p.ns * KEYS >= p.lo) p.ns = p.lo = 0;  // the two meet
    const int tiles = p.ns + (p.end - p.lo + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
    p.i0 = min(p.sp * per, tiles);
    p.i1 = min(p.i0 + per, tiles);
    p.ok = true;
    return p;
}
template <int KEYS>
__device__ __forceinline__ int tile_key(const RowsPlace &p, int i) {
    return i < p.ns ? i * KEYS : p.lo + (i - p.ns) * KEYS;
}

// Whether the row at position p sees key j.
__device__ __forceinline__ bool sees(const RowsArgs &a, int p, int j) {
    return j <= p && (a.window == 0 || j > p - a.window || j < a.sink);
}
// Whether all rows at positions p0..p1 see all keys j0..j1, and whether none sees any.
__device__ __forceinline__ bool all_see(const RowsArgs &a, int p0, int p1, int j0, int j1) {
    return j1 <= p0 && (a.window == 0 || j0 > p1 - a.window || j1 < a.sink);
}
__device__ __forceinline__ bool none_sees(const RowsArgs &a, int p0, int p1, int j0, int j1) {
    return j0 > p1 || (a.window != 0 && j1 <= p0 - a.window && j0 >= a.sink);
}

// The pool row of row j of stream b. Pages outside the pool read page 0.
__device__ __forceinline__ int pool_row(const RowsArgs &a, int b, int j) {
    int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + (j >> a.c.shift)];
    if (pg < 0 || pg >= a.c.pool_pages) pg = 0;
    return (pg << a.c.shift) + (j & ((1 << a.c.shift) - 1));
}

__device__ __forceinline__ float half_value(uint16_t h, int type) {
    return type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}
// Value i of an array of float32, float16 or bfloat16, widened.
__device__ __forceinline__ float load_any(const void *p, int type, long long i) {
    return type == 0 ? static_cast<const float *>(p)[i] : half_value(static_cast<const uint16_t *>(p)[i], type);
}
__device__ __forceinline__ void store_any(void *p, int type, long long i, float x) {
    if (type == 0)
        static_cast<float *>(p)[i] = x;
    else if (type == 1)
        static_cast<_Float16 *>(p)[i] = static_cast<_Float16>(x);
    else
        static_cast<__bf16 *>(p)[i] = static_cast<__bf16>(x);
}
// Value d of a cache row's head, without its scale.
__device__ __forceinline__ float cache_value(const unsigned char *row, int type, int d) {
    if (type <= 2) return load_any(row, type, d);
    return type == 4 ? __builtin_amdgcn_cvt_f32_fp8(row[d], 0) : static_cast<float>(static_cast<int8_t>(row[d]));
}

// Columns c of `mask` (first column col0) again, key by key, by one wavefront:
// lane j of 64 keys has its logit, then lane d its values. The largest weight is
// 1. Rare (a NaN or a sum past kMostSum among the outputs), so plain.
template <int KEYS>
__device__ __forceinline__ void repair_columns(const RowsArgs &a, const RowsPlace &p, int col0, unsigned mask) {
    const int lane = threadIdx.x & 63;
    const unsigned char *kp = a.c.k + static_cast<long long>(p.h) * a.k_head, *vp = a.c.v + static_cast<long long>(p.h) * a.v_head;
    while (mask) {
        const int c = __ffs(mask) - 1;
        mask &= mask - 1;
        const int col = col0 + c, row = col / a.group, head = p.h * a.group + col % a.group, at = p.pos + row;
        const long long qo = static_cast<long long>(p.b) * a.q_stream + static_cast<long long>(row) * a.q_row +
                             static_cast<long long>(head) * a.c.qk;
        bool nan = false;  // of the query: the outputs are NaN as they stand
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < a.c.qk) nan |= isnan(load_any(a.q, a.type, qo + lane + 64 * e));
        if (__any(nan)) continue;
        float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = p.i0; i < p.i1; ++i)
            for (int j0 = tile_key<KEYS>(p, i), j1 = j0 + KEYS; j0 < j1; j0 += 64) {
                const int j = j0 + lane;
                const bool seen = lane < KEYS && sees(a, at, j);
                float x = -INFINITY, vs = 1.0f;
                int r = 0;
                if (seen) {
                    r = pool_row(a, p.b, j);
                    const unsigned char *k = kp + static_cast<long long>(r) * a.k_row;
                    x = 0.0f;
                    for (int d = 0; d < a.c.qk; ++d) x = fmaf(load_any(a.q, a.type, qo + d), cache_value(k, a.c.type, d), x);
                    if (a.c.type >= 3) {
                        const long long sat = static_cast<long long>(r >> a.c.sshift) * a.c.kv_heads + p.h;
                        x *= a.c.ks[sat];
                        vs = a.c.vs[sat];
                    }
                    x *= a.scale_log2;
                }
                float mt = x;
#pragma unroll
                for (int s = 32; s > 0; s >>= 1) mt = fmaxf(mt, xor_lane(mt, s));
                const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.0f : mn;
                const float f = __builtin_amdgcn_exp2f(m - mu);
                m = mn;
                l *= f;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= f;
                const float w = seen ? __builtin_amdgcn_exp2f(x - mu) : 0.0f;
                l += w;
                unsigned long long live = __ballot(seen);
                while (live) {
                    const int k = __ffsll(live) - 1;
                    live &= live - 1;
                    const float wk = __shfl(w, k) * __shfl(vs, k);
                    const unsigned char *v = vp + static_cast<long long>(__shfl(r, k)) * a.v_row;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (lane + 64 * e < a.c.vd) o[e] = fmaf(wk, cache_value(v, a.c.type, lane + 64 * e), o[e]);
                }
            }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) l += xor_lane(l, s);
        if (a.part) {
            const long long pi = ((static_cast<long long>(p.b) * a.t + row) * a.heads + head) * a.splits + p.sp;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < a.c.vd) a.part[pi * a.c.vd + lane + 64 * e] = o[e];
            if (lane == 0) {
                a.part_ml[2 * pi] = m;
                a.part_ml[2 * pi + 1] = l;
            }
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const long long to = static_cast<long long>(p.b) * a.out_stream + static_cast<long long>(row) * a.out_row +
                                 static_cast<long long>(head) * a.c.vd;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < a.c.vd) store_any(a.out, a.type, to + lane + 64 * e, o[e] * inv);
        }
    }
}

template <class F>
hipError_t launch_with(F *fn, const RowsArgs &a, int wg_cols, int lds, std::atomic<unsigned long long> &attr, hipStream_t s) {
    if (lds > 64 * 1024)
        if (hipError_t e = lds_limit_once(reinterpret_cast<const void *>(fn), lds, attr)) return e;
    const int cols = a.t * a.group, col_tiles = (cols + wg_cols - 1) / wg_cols;
    const long long per = static_cast<long long>(col_tiles) * a.splits, each = 8 / std::min(8, a.c.kv_heads);
    const long long grid = rows_by_head(a) ? (per + each - 1) / each * 8 * a.batch
                                           : xcd_grid(static_cast<long long>(a.batch) * a.c.kv_heads, per);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(64 * kRWaves), lds, s, a, col_tiles);
    return hipGetLastError();
}

}  // namespace cqhip
