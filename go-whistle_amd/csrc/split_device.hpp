// What the kernels of split_kernels.hip and parts_kernels.hip share: the values
// of a piece of a row, a list's keys and its parts, and the join of a
// workgroup's wavefronts.
#pragma once

#include "cq_internal.hpp"
#include "cq_device.hpp"

namespace cqhip {

using f32x4 = float __attribute__((ext_vector_type(4)));

constexpr int kCols = 16;
constexpr size_t kMostLds = 150 * 1024;

// The e-th value of a lane's piece of a row, as float32.
template <int TYPE>
__device__ __forceinline__ float piece_value(const uint32_t *w, int e) {
    if constexpr (TYPE == 0) {
        return __uint_as_float(w[e]);
    } else if constexpr (TYPE == 1) {
        const uint16_t h = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
        return static_cast<float>(__builtin_bit_cast(_Float16, h));
    } else if constexpr (TYPE == 2) {
        return __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
    } else if constexpr (TYPE != 4) {
        return static_cast<float>(static_cast<int32_t>(w[e >> 2] << (24 - 8 * (e & 3))) >> 24);
    } else {
        const int x = static_cast<int>(w[e >> 2]);
        switch (e & 3) {  // the byte is an immediate
            case 0: return __builtin_amdgcn_cvt_f32_fp8(x, 0);
            case 1: return __builtin_amdgcn_cvt_f32_fp8(x, 1);
            case 2: return __builtin_amdgcn_cvt_f32_fp8(x, 2);
            default: return __builtin_amdgcn_cvt_f32_fp8(x, 3);
        }
    }
}

// The cache types: float32, float16, bfloat16, then codes of 8 bits with
// scales: int8 (a scale a row), e4m3 and int8 (a scale a page).
template <int TYPE>
constexpr bool kScaled = TYPE >= 3;
template <int TYPE>
constexpr bool kFinite = TYPE == 3 || TYPE == 5;  // every code is
template <int TYPE>
constexpr int kValueSize = TYPE == 0 ? 4 : kScaled<TYPE> ? 1 : 2;

// Where the scales of an 8-bit row are.
__device__ __forceinline__ long long scale_at(const SplitArgs &a, long long row, int h) {
    return (row >> a.c.sshift) * a.c.kv_heads + h;
}

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t *w, const unsigned char *p) {
    if constexpr (WORDS >= 4) {
#pragma unroll
        for (int k = 0; k < WORDS; k += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + 4 * k);
            w[k] = x.x;
            w[k + 1] = x.y;
            w[k + 2] = x.z;
            w[k + 3] = x.w;
        }
    } else if constexpr (WORDS == 2) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x;
        w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// Value i of an array of `type` (float32, float16, bfloat16), widened.
__device__ __forceinline__ float load_value(const void *p, int type, long long i) {
    if (type == 0) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// Stored to the nearest even.
__device__ __forceinline__ void store_value(void *p, int type, long long i, float x) {
    if (type == 0)
        static_cast<float *>(p)[i] = x;
    else if (type == 1)
        static_cast<_Float16 *>(p)[i] = static_cast<_Float16>(x);
    else
        static_cast<__bf16 *>(p)[i] = static_cast<__bf16>(x);
}

// A stream's rows' count: of causal rows none where they do not lie inside the cache.
__device__ __forceinline__ int q_rows(const SplitArgs &a, int b) {
    if (a.pos) {
        const int n = a.q_len ? a.q_len[b] : a.t, p = a.pos[b];
        return n <= 0 || n > a.t || p < 0 || p > a.nk_max - n ? 0 : n;
    }
    return a.q_len ? min(max(a.q_len[b], 0), a.t) : a.t;
}

// The keys of a stream: two spans of row numbers, or the first n rows of a
// memory; of causal rows first..last those that any of them sees.
struct KeyList {
    int lo0, n0, lo1, n;
    bool ok;
    __device__ int row(int j) const { return j < n0 ? lo0 + j : lo1 + (j - n0); }
};

__device__ __forceinline__ KeyList key_list(const SplitArgs &a, int b, int mem, int first = 0, int last = 0) {
    KeyList l{0, 0, 0, 0, true};
    if (a.pos) {
        const int p = a.pos[b];
        l.lo1 = a.window ? max(p + first - a.window + 1, 0) : 0;
        l.n0 = a.window ? min(a.sink, l.lo1) : 0;
        l.n = l.n0 + (p + last + 1 - l.lo1);
    } else if (a.spans) {
        const int32_t *sp = a.spans + static_cast<long long>(b) * 4;
        const int lo0 = sp[0], hi0 = sp[1], lo1 = sp[2], hi1 = sp[3];
        l.ok = lo0 >= 0 && lo0 <= hi0 && hi0 <= a.nk_max && lo1 >= 0 && lo1 <= hi1 && hi1 <= a.nk_max &&
               (hi0 <= lo1 || hi0 == lo0 || hi1 == lo1);
        l.lo0 = lo0;
        l.n0 = hi0 - lo0;
        l.lo1 = lo1;
        l.n = l.n0 + (hi1 - lo1);
    } else {
        l.ok = mem >= 0 && mem < a.memories;
        l.n = a.k_len && l.ok ? min(max(a.k_len[mem], 0), a.nk_max) : a.nk_max;
        l.n0 = l.n;
    }
    if (!l.ok) l.n = 0;
    return l;
}

// Keys a part of the list takes: whole tiles of 64 keys, equal over the parts.
__device__ __forceinline__ int part_keys(int n, int splits) {
    const int units = (n + 63) / 64;
    return (units + splits - 1) / splits * 64;
}

// The causal stream with the place-th longest list (up to 64 streams). A launch of
// several rounds of workgroups takes the long ones first, so that none begins as
// the last ones end, and neighbours, which go to different XCDs, are alike (5
// drafts of 32 streams of up to 8000 e4m3 keys: 101 -> 95 us).
__device__ __forceinline__ int longest_stream(const SplitArgs &a, int place) {
    const int lane = threadIdx.x & 63;
    int n = -1;
    if (lane < a.batch) {
        const int rows = q_rows(a, lane);
        n = rows ? a.pos[lane] + rows : 0;
    }
    int rank = 0;
    for (int b = 0; b < a.batch; ++b) {
        const int other = __builtin_amdgcn_readlane(n, b);
        rank += other > n || (other == n && b < lane);
    }
    return __ffsll(__ballot(lane < a.batch && rank == place)) - 1;
}

// What a workgroup works on.
struct Place {
    int sp, ct, h, b, mem, group, cols, j0, j1;
    int pos0, pos1;  // causal: the positions of the tile's first and last rows
    KeyList kl;
    bool ok;
};
__device__ __forceinline__ Place place_of(const SplitArgs &a, int col_tiles, int tile_cols) {
    Place p;
    // A part's key heads on one XCD: rows of narrow heads share cache lines
    // (256 streams of 448 int8 keys, 8 heads of 64, spread over the XCDs 32.8
    // us: every line, and the scales' eight times, was read more than once).
    const XcdPlace x = xcd_place(a.batch * a.splits, a.c.kv_heads * col_tiles);
    p.ct = p.sp = 0;
    p.h = x.within;
    if (col_tiles > 1) {
        p.h = x.within / col_tiles;
        p.ct = x.within - p.h * col_tiles;
    }
    p.b = x.unit;
    if (a.splits > 1) {
        p.b = x.unit / a.splits;
        p.sp = x.unit - p.b * a.splits;
    }
    if (!x.ok) {
        p.ok = false;
        return p;
    }
    if (a.by_length) p.b = longest_stream(a, p.b);
    p.group = a.group;
    p.mem = a.index ? a.index[p.b] : p.b;
    p.cols = q_rows(a, p.b) * p.group;
    if (a.pos) {
        const int first = p.ct * tile_cols / p.group, last = (min(p.ct * tile_cols + tile_cols, p.cols) - 1) / p.group;
        p.pos0 = a.pos[p.b] + first;
        p.pos1 = a.pos[p.b] + last;
        p.kl = key_list(a, p.b, p.mem, first, last);
    } else {
        p.kl = key_list(a, p.b, p.mem);
    }
    p.ok = p.kl.ok && p.ct * tile_cols < p.cols;
    p.j0 = 0;
    p.j1 = p.kl.n;
    if (a.splits > 1) {
        const int per = part_keys(p.kl.n, a.splits);
        p.j0 = min(p.sp * per, p.kl.n);
        p.j1 = min(p.j0 + per, p.kl.n);
    }
    return p;
}

// Column cn's query row and head.
__device__ __forceinline__ void column_of(const SplitArgs &a, const Place &p, int cn, int &row, int &head) {
    row = a.t == 1 ? 0 : cn / p.group;
    head = p.h * p.group + cn - row * p.group;
}
__device__ __forceinline__ long long query_at(const SplitArgs &a, const Place &p, int cn) {
    int row, head;
    column_of(a, p, cn, row, head);
    return static_cast<long long>(p.b) * a.q_stream + static_cast<long long>(row) * a.q_row +
           static_cast<long long>(head) * a.c.qk;
}
__device__ __forceinline__ long long part_at(const SplitArgs &a, const Place &p, int row, int head) {
    return ((static_cast<long long>(p.b) * a.t + row) * a.heads + head) * a.splits + p.sp;
}

// Over the 16 lanes of a row, in all of them.
template <int N>
__device__ __forceinline__ float rotated(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_sum(float x) {
    x += rotated<8>(x);
    x += rotated<4>(x);
    x += rotated<2>(x);
    return x + rotated<1>(x);
}
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, rotated<8>(x));
    x = fmaxf(x, rotated<4>(x));
    x = fmaxf(x, rotated<2>(x));
    return fmaxf(x, rotated<1>(x));
}

// The pool (or memory) row of key j of the list.
__device__ __forceinline__ int array_row(const SplitArgs &a, const Place &p, int j) {
    const int row = p.kl.row(j);
    if (!a.c.pages) return row;
    int pg = a.c.pages[static_cast<long long>(p.b) * a.c.page_stride + (row >> a.c.shift)];
    if (pg < 0 || pg >= a.c.pool_pages) pg = 0;
    return (pg << a.c.shift) + (row & ((1 << a.c.shift) - 1));
}

// N consecutive query values from element i on (VEC: pieces of four are aligned to their size).
template <int N, bool VEC>
__device__ __forceinline__ void load_query_values(float *x, const SplitArgs &a, long long i) {
    if constexpr (VEC) {
        if (a.type == 0) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + i + e);
                x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
            }
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int e = 0; e < N; e += 4)
                *reinterpret_cast<uint2 *>(w + e / 2) =
                    *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + i + e);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = a.type == 1 ? piece_value<1>(w, e) : piece_value<2>(w, e);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = load_value(a.q, a.type, i + e);
    }
}
// The same, times f.
template <int N>
__device__ __forceinline__ void load_query(float *x, const SplitArgs &a, long long i, float f) {
    if (a.q_vec)
        load_query_values<N, true>(x, a, i);
    else
        load_query_values<N, false>(x, a, i);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] *= f;
}

// LDS of a workgroup, in floats: per wavefront and column the maximum and the
// sum, per column the joined maximum and 1 / sum, then from a 16-byte boundary
// per wavefront and column the outputs (rows of D + 4), then the logits
// [column][nk_max] where the weights are asked of a whole list.
template <int COLS, int D>
struct Joint {
    static constexpr int kRow = D + 4;
    float *ml, *stat, *o, *logits;
    static constexpr int stats(int waves) { return (waves * 2 * COLS + 2 * COLS + 3) / 4 * 4; }
    static constexpr int floats(int waves) { return stats(waves) + waves * COLS * kRow; }
    static constexpr bool aligned() {  // the outputs' rows, stored as float4, for every number of wavefronts
        for (int w = 1; w <= 8; ++w)
            if (stats(w) % 4 != 0) return false;
        return kRow % 4 == 0;
    }
    __device__ Joint(float *smem, int waves)
        : ml(smem), stat(ml + waves * 2 * COLS), o(smem + stats(waves)), logits(smem + floats(waves)) {
        static_assert(aligned(), "outputs off their 16-byte boundary");
    }
};

// Whether the row at position p sees row j.
__device__ __forceinline__ bool sees_row(const SplitArgs &a, int p, int j) {
    return (j <= p) & ((a.window == 0) | (j > p - a.window) | (j < a.sink));  // no branches
}

// A column again, key by key, by one wavefront: lane j of 64 keys has its logit,
// then lane d its values. A key that a causal column does not see has the weight 0,
// and 0 times an infinite or NaN value is NaN, as are parts of a weight times an
// infinity; and sums past kMostSum may have weights of 2^8: columns that come out
// so are computed here, which skips what they do not see, with weights up to 1. Rare, so
// plain. Returns value d = lane + 64 e in o[e].
// false, and nothing, of a query that holds a NaN, whose outputs are NaN as they stand.
template <int TYPE>
__device__ __forceinline__ bool repair_column(const SplitArgs &a, const Place &p, int row, int head, float &m, float &l,
                                              float (&o)[4]) {
    const int lane = threadIdx.x & 63, at = a.pos ? a.pos[p.b] + row : 0;
    const long long qo = static_cast<long long>(p.b) * a.q_stream + static_cast<long long>(row) * a.q_row +
                         static_cast<long long>(head) * a.c.qk;
    const unsigned char *kp = a.c.k + static_cast<long long>(p.h) * a.k_head, *vp = a.c.v + static_cast<long long>(p.h) * a.v_head;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.c.qk) nan |= isnan(load_value(a.q, a.type, qo + lane + 64 * e));
    if (__any(nan)) return false;
    m = -INFINITY;
    l = o[0] = o[1] = o[2] = o[3] = 0.0f;
    auto value = [&](const unsigned char *r, int d) {
        constexpr int kWordValues = 4 / kValueSize<TYPE>;
        const uint32_t w = reinterpret_cast<const uint32_t *>(r)[d / kWordValues];
        if constexpr (kScaled<TYPE>) {  // the byte is an immediate
            const uint32_t x = w >> (8 * (d & 3));
            return piece_value<TYPE>(&x, 0);
        } else {
            return TYPE == 0 ? piece_value<TYPE>(&w, 0) : piece_value<TYPE>(&w, d & 1);
        }
    };
    for (int j0 = p.j0; j0 < p.j1; j0 += 64) {
        const int j = j0 + lane;
        const bool seen = j < p.j1 && (!a.pos || sees_row(a, at, p.kl.row(j)));
        float x = -INFINITY, vs = 1.0f;
        int r = 0;
        if (seen) {
            r = array_row(a, p, j);
            const unsigned char *k = kp + static_cast<long long>(r) * a.k_row;
            x = 0.0f;
            for (int d = 0; d < a.c.qk; ++d) x = fmaf(load_value(a.q, a.type, qo + d), value(k, d), x);
            if constexpr (kScaled<TYPE>) {
                x *= a.c.ks[scale_at(a, r, p.h)];
                vs = a.c.vs[scale_at(a, r, p.h)];
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
                if (lane + 64 * e < a.c.vd) o[e] = fmaf(wk, value(v, lane + 64 * e), o[e]);
        }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) l += xor_lane(l, s);
    return true;
}

// Joins the wavefronts' columns (o, ml filled, outputs relative to each
// wavefront's own maximum) and writes them: the outputs, or a part's sums.
// TYPE: the cache's type where columns may have to be computed again, else -1.
template <int COLS, int D, int TYPE = -1>
__device__ __forceinline__ void finish(const SplitArgs &a, const Place &p, const Joint<COLS, D> &jt) {
    const int tid = threadIdx.x, threads = blockDim.x, waves = threads >> 6;
    const int col0 = p.ct * COLS, nc = min(COLS, p.cols - col0);
    __syncthreads();
    if (tid < nc) {
        float mx = -INFINITY, sum = 0.0f;
        for (int w = 0; w < waves; ++w) mx = fmaxf(mx, jt.ml[(w * 2) * COLS + tid]);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        for (int w = 0; w < waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(jt.ml[(w * 2) * COLS + tid] - mu);
            sum += jt.ml[(w * 2 + 1) * COLS + tid] * f;
            jt.ml[(w * 2) * COLS + tid] = f;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        jt.stat[tid] = mu;
        jt.stat[COLS + tid] = inv;
        if (a.part) {
            int row, head;
            column_of(a, p, col0 + tid, row, head);
            const long long pi = part_at(a, p, row, head);
            a.part_ml[2 * pi] = mx;
            a.part_ml[2 * pi + 1] = sum;
        }
    }
    __syncthreads();
    for (int n = tid >> 6; n < nc; n += waves) {
        int row, head;
        column_of(a, p, col0 + n, row, head);
        bool again = false;
        for (int d = tid & 63; d < a.c.vd; d += 64) {
            float v = 0.0f;
            for (int w = 0; w < waves; ++w) v = fmaf(jt.o[(w * COLS + n) * jt.kRow + d], jt.ml[(w * 2) * COLS + n], v);
            again |= !(fabsf(v) < kMostSum);
            if (a.part)
                a.part[part_at(a, p, row, head) * a.c.vd + d] = v;
            else
                store_value(a.out, a.type,
                            static_cast<long long>(p.b) * a.out_stream + static_cast<long long>(row) * a.out_row +
                                static_cast<long long>(head) * a.c.vd + d,
                            v * jt.stat[COLS + n]);
        }
        if constexpr (TYPE >= 0) {
            if (!__any(again)) continue;
            float m, l, o[4];
            if (!repair_column<TYPE>(a, p, row, head, m, l, o)) continue;
            const float inv = a.part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const long long pi = part_at(a, p, row, head);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = (tid & 63) + 64 * e;
                if (d >= a.c.vd) continue;
                if (a.part)
                    a.part[pi * a.c.vd + d] = o[e];
                else
                    store_value(a.out, a.type,
                                static_cast<long long>(p.b) * a.out_stream + static_cast<long long>(row) * a.out_row +
                                    static_cast<long long>(head) * a.c.vd + d,
                                o[e] * inv);
            }
            if (a.part && (tid & 63) == 0) {
                a.part_ml[2 * pi] = m;
                a.part_ml[2 * pi + 1] = l;
            }
        }
    }
    if (a.acc_out && !a.logits) {  // the whole list's weights
        for (int j = tid; j < p.kl.n; j += threads) {
            float w = 0.0f;
            for (int n = 0; n < nc; ++n)
                w += __builtin_amdgcn_exp2f(jt.logits[n * a.nk_max + j] - jt.stat[n]) * jt.stat[COLS + n];
            const long long at = (static_cast<long long>(p.b) * a.c.kv_heads + p.h) * a.acc_cap + p.kl.row(j);
            a.acc_out[at] = (a.acc ? a.acc[at] : 0.0f) + w;
        }
    }
}

// Two floats' upper halves: x in the lower 16 bits, y in the upper.
__device__ __forceinline__ uint32_t upper_pair(float x, float y) {
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
}

template <int TYPE>
__device__ __forceinline__ f32x4 mfma_16x16x32(const uint32_t *a, const uint32_t *b, f32x4 c) {
    using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
    const u32x4 x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
    if constexpr (TYPE == 1) {
        using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    } else {
        using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    }
}

// LDS of a launch, in bytes: the joint of its wavefronts and the logits.
template <int COLS, int D>
size_t joint_lds(const SplitArgs &a, int waves) {
    const size_t lg = a.acc_out && !a.logits ? static_cast<size_t>(a.heads / a.c.kv_heads) * a.nk_max : 0;
    return sizeof(float) * (Joint<COLS, D>::floats(waves) + lg);
}

template <class F>
hipError_t launch_with(F *fn, const SplitArgs &a, int tile_cols, size_t lds, std::atomic<unsigned long long> &attr, hipStream_t s) {
    if (lds > 64 * 1024)
        if (hipError_t e = lds_limit_once(reinterpret_cast<const void *>(fn), kMostLds, attr)) return e;
    const int cols = a.t * (a.heads / a.c.kv_heads), col_tiles = (cols + tile_cols - 1) / tile_cols;
    const long long grid = xcd_grid(static_cast<long long>(a.batch) * a.splits, static_cast<long long>(a.c.kv_heads) * col_tiles);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(64 * a.waves), lds, s, a, col_tiles);
    return hipGetLastError();
}

}  // namespace cqhip
