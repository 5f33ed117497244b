// gfx950 kernels that write paged caches of any type: the append of new rows
// (kv_append_paged_dev) and the eviction by accumulated weight
// (kv_evict_paged_dev).
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

// ---- append ---------------------------------------------------------------------

// A head's row of width values is one unit: LANES = the power of two of lanes
// that hold it at four values each, so a wavefront takes 64 / LANES units and
// an int8 row's bound is a few exchanges within them. Units in (keys or
// values, stream, row, head) order: a wavefront's loads and stores are
// consecutive.
template <int TYPE, int LANES>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, long long units, int vec) {
    const long long u = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / LANES;
    if (u >= 2 * units) return;
    const int which = u >= units;
    const long long w = which ? u - units : u;
    const int h = static_cast<int>(w % a.c.kv_heads);
    const long long bi = w / a.c.kv_heads;
    const int i = static_cast<int>(bi % a.t), b = static_cast<int>(bi / a.t);
    if (a.rows) {
        const int n = a.rows[b];
        if (n > a.t || i >= n) return;
    }
    const long long p = static_cast<long long>(a.pos[b]) + i;
    if (p < 0 || p >= a.cap) return;
    const int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + (p >> a.c.shift)];
    if (pg < 0 || pg >= a.c.pool_pages) return;
    const long long row = (static_cast<long long>(pg) << a.c.shift) + (p & ((1 << a.c.shift) - 1));
    const int width = which ? a.c.vd : a.c.qk;
    const int lane = threadIdx.x & (LANES - 1), d = 4 * lane;
    if (a.acc && !which && lane == 0) a.acc[(static_cast<long long>(b) * a.c.kv_heads + h) * a.acc_cap + p] = 0.0f;
    const long long at = static_cast<long long>(b) * a.stream[which] + static_cast<long long>(i) * a.row[which] +
                         static_cast<long long>(h) * width + d;
    const bool live = d < width;
    float x[4] = {0, 0, 0, 0};
    if (live) {
        if (a.type == 0) {
            const float *s = static_cast<const float *>(a.x[which]) + at;
            if (vec >> which & 1) {
                const float4 v = *reinterpret_cast<const float4 *>(s);
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = s[e];
            }
        } else {
            const uint16_t *s = static_cast<const uint16_t *>(a.x[which]) + at;
            uint16_t v[4];
            if (vec >> which & 1) {
                *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(s);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = s[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = a.type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, v[e]))
                                   : __uint_as_float(static_cast<uint32_t>(v[e]) << 16);
        }
    }
    unsigned char *dst = which ? a.c.v : a.c.k;
    const long long to = (row * a.c.kv_heads + h) * width + d;
    if constexpr (TYPE == 3) {
        // QuantizeRow (int8.go:36-55) over the head's values
        float m = go_max(go_max(fabsf(x[0]), fabsf(x[1])), go_max(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = go_max(m, __shfl_xor(m, o));
        const float sc = m > 0.0f ? m / 127.0f : 1.0f;
        if (live) {
            uint32_t q = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) q |= (static_cast<uint32_t>(go_int8_code(rintf(x[e] / sc))) & 255u) << (8 * e);
            *reinterpret_cast<uint32_t *>(dst + to) = q;
        }
        if (lane == 0) (which ? a.c.vs : a.c.ks)[row * a.c.kv_heads + h] = sc;
    } else if (live) {
        if constexpr (TYPE == 0) {
            reinterpret_cast<float4 *>(dst)[to >> 2] = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            uint16_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = TYPE == 1 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[e]))
                                 : __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[e]));
            reinterpret_cast<uint2 *>(dst)[to >> 2] = *reinterpret_cast<uint2 *>(v);
        }
    }
}

template <int TYPE, int LANES>
hipError_t launch_append_lanes(const PagedAppendArgs &a, int vec, hipStream_t s) {
    const long long units = static_cast<long long>(a.batch) * a.t * a.c.kv_heads;
    const long long blocks = (2 * units * LANES + 255) / 256;
    hipLaunchKernelGGL((paged_append_kernel<TYPE, LANES>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a,
                       units, vec);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_append_type(const PagedAppendArgs &a, int vec, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return launch_append_lanes<TYPE, 16>(a, vec, s);
    if (w <= 128) return launch_append_lanes<TYPE, 32>(a, vec, s);
    return launch_append_lanes<TYPE, 64>(a, vec, s);
}

// ---- eviction -------------------------------------------------------------------

constexpr int kSelThreads = 1024;

// A weight's place in the order of weights: larger is kept sooner. Held rows
// (the first sink, the last recent) come before every weight; -0 is 0; a NaN
// is the least.
__device__ __forceinline__ uint32_t weight_key(float w, bool held) {
    if (held) return 0xffffffffu;
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// The sum of v over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int scan_before(int v, int *sh, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 63) sh[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < kSelThreads / 64; ++w) {
        if (w < wave) before += sh[w];
        total += sh[w];
    }
    return before + s - v;
}

// The kept rows of one (stream, key head): the keep-th largest key by a radix
// selection of four 8-bit digits (a 256-entry histogram in LDS each), then
// one ordered pass that writes the rows above it, and the lowest of those
// equal to it, in row order. Integer counts throughout: the same rows in
// every run.
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int scan_sh[kSelThreads / 64];
    __shared__ int digit_sh, need_sh;
    const int tid = threadIdx.x;
    const int h = blockIdx.x % a.c.kv_heads, b = blockIdx.x / a.c.kv_heads;
    const int n = a.len[b];
    if (n < 0 || n > a.nk_max) return;
    const long long bh = static_cast<long long>(b) * a.c.kv_heads + h;
    const float *w = a.acc + bh * a.acc_cap;
    int32_t *kept = a.kept + bh * a.keep;
    float *out = a.acc_out + bh * a.acc_out_cap;
    const int live = min(n, a.keep);
    for (int i = live + tid; i < a.keep; i += kSelThreads) kept[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += kSelThreads) {
            kept[i] = i;
            out[i] = w[i];
        }
        return;
    }
    if (a.keep == 0) return;
    auto key_of = [&](int j) { return weight_key(w[j], j < a.sink || j >= n - a.recent); };
    // the keep-th largest key, and how many of the rows that equal it are kept
    uint32_t thr = 0;
    int need = a.keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += kSelThreads) {
            const uint32_t k = key_of(j);
            if (shift == 24 || (k >> (shift + 8)) == (thr >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int left = need, d = 255;
            while (d > 0 && hist[d] < left) left -= hist[d--];
            digit_sh = d;
            need_sh = left;
        }
        __syncthreads();
        thr |= static_cast<uint32_t>(digit_sh) << shift;
        need = need_sh;
        __syncthreads();
    }
    // each thread a run of rows
    const int per = (n + kSelThreads - 1) / kSelThreads;
    const int r0 = min(tid * per, n), r1 = min(r0 + per, n);
    int above = 0, equal = 0;
    for (int j = r0; j < r1; ++j) {
        const uint32_t k = key_of(j);
        above += k > thr;
        equal += k == thr;
    }
    int total;
    int eq = scan_before(equal, scan_sh, total);
    const int kept_eq = max(0, min(equal, need - eq));
    int at = scan_before(above + kept_eq, scan_sh, total);
    for (int j = r0; j < r1; ++j) {
        const uint32_t k = key_of(j);
        if (k > thr || (k == thr && eq++ < need)) {
            kept[at] = j;
            out[at] = w[j];
            ++at;
        }
    }
}

// The kept rows copied: 16 bytes a thread, pieces of a head's key row, then of
// its value row; row i of every head of a stream side by side, so a
// destination row is written whole. The scales of int8 rows ride with the
// first piece. Also the streams' new lengths.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a, int kpieces, int pieces, long long total) {
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (id < a.batch) {
        const int n = a.len[id];
        if (n >= 0 && n <= a.nk_max) a.len_out[id] = min(n, a.keep);
    }
    if (id >= total) return;
    const int per_row = pieces * a.c.kv_heads;
    const long long bi = id / per_row;
    const int x = static_cast<int>(id - bi * per_row);
    const int i = static_cast<int>(bi % a.keep), b = static_cast<int>(bi / a.keep);
    const int n = a.len[b];  // or already its new value: in [0, nk_max] both or neither
    if (n < 0 || n > a.nk_max) return;
    const bool val = x >= kpieces * a.c.kv_heads;  // a row's keys of all heads, then its values
    const int np = val ? pieces - kpieces : kpieces;
    const int y = val ? x - kpieces * a.c.kv_heads : x;
    const int h = y / np, p = y - h * np;
    const int j = a.kept[(static_cast<long long>(b) * a.c.kv_heads + h) * a.keep + i];
    if (j < 0) return;
    int sp = a.c.pages[static_cast<long long>(b) * a.c.page_stride + (j >> a.c.shift)];
    if (sp < 0 || sp >= a.c.pool_pages) sp = 0;
    const int dp = a.dst_pages[static_cast<long long>(b) * a.dst_stride + (i >> a.c.shift)];
    if (dp < 0 || dp >= a.c.pool_pages) return;
    const int mask = (1 << a.c.shift) - 1;
    const long long from = ((static_cast<long long>(sp) << a.c.shift) + (j & mask)) * a.c.kv_heads + h;
    const long long to = ((static_cast<long long>(dp) << a.c.shift) + (i & mask)) * a.c.kv_heads + h;
    uint4 *pool = reinterpret_cast<uint4 *>(val ? a.c.v : a.c.k);
    pool[to * np + p] = pool[from * np + p];
    if (a.c.type == 3 && p == 0) {
        float *s = val ? a.c.vs : a.c.ks;
        s[to] = s[from];
    }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t s) {
    int vec = 0;  // the rows' four-value pieces are aligned to their size
    const int size = a.type == 0 ? 4 : 2;
    for (int k = 0; k < 2; ++k)
        if ((reinterpret_cast<uintptr_t>(a.x[k]) | (a.stream[k] * size) | (a.row[k] * size)) % (4 * size) == 0) vec |= 1 << k;
    switch (a.c.type) {
        case 0: return launch_append_type<0>(a, vec, s);
        case 1: return launch_append_type<1>(a, vec, s);
        case 2: return launch_append_type<2>(a, vec, s);
        default: return launch_append_type<3>(a, vec, s);
    }
}

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(static_cast<unsigned>(a.batch) * a.c.kv_heads), dim3(kSelThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int size = a.c.type == 0 ? 4 : a.c.type == 3 ? 1 : 2;
    const int kpieces = a.c.qk * size / 16, pieces = kpieces + a.c.vd * size / 16;
    const long long total = static_cast<long long>(a.batch) * a.keep * a.c.kv_heads * pieces;
    const long long blocks = (std::max<long long>(total, a.batch) + 255) / 256;
    hipLaunchKernelGGL(evict_copy_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, kpieces, pieces, total);
    return hipGetLastError();
}

}  // namespace cqhip
