// gfx950 kernels that write paged caches of any type: the append of new rows
// (kv_append_paged_dev) and the eviction by accumulated weight
// (kv_evict_paged_dev).
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

// ---- append ---------------------------------------------------------------------

// Four values of a row, from an array of `type` (vec: its pieces of four are
// aligned to their size), widened.
__device__ __forceinline__ void load_four(float *x, const void *p, int type, long long at, bool vec) {
    if (type == 0) {
        const float *s = static_cast<const float *>(p) + at;
        if (vec) {
            const float4 u = *reinterpret_cast<const float4 *>(s);
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = s[e];
        }
        return;
    }
    const uint16_t *s = static_cast<const uint16_t *>(p) + at;
    uint32_t w[2];
    if (vec) {
        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(s);
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) w[e] = s[2 * e] | static_cast<uint32_t>(s[2 * e + 1]) << 16;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t h = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        x[e] = type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
    }
}

// A head's key row and value row of one stream's row are one unit: LANES = the
// power of two of lanes that hold a row at four values each, so a wavefront
// takes 64 / LANES units, the way through the page table is paid once for
// both rows, and an int8 row's bound is a few exchanges within its lanes.
// Units in (stream, row, head) order: a wavefront's loads and stores are
// consecutive.
template <int TYPE, int LANES>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, unsigned units, int vec) {
    const unsigned u = (blockIdx.x * 256u + threadIdx.x) / LANES;
    if (u >= units) return;
    const unsigned bi = u / a.c.kv_heads;
    const int h = static_cast<int>(u - bi * a.c.kv_heads);
    const int b = static_cast<int>(bi / a.t), i = static_cast<int>(bi - static_cast<unsigned>(b) * a.t);
    if (a.rows) {
        const int n = a.rows[b];
        if (n > a.t || i >= n) return;
    }
    const long long p = static_cast<long long>(a.pos[b]) + i;
    if (p < 0 || p >= a.cap) return;
    const int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + (p >> a.c.shift)];
    if (pg < 0 || pg >= a.c.pool_pages) return;
    const long long to = ((static_cast<long long>(pg) << a.c.shift) + (p & ((1 << a.c.shift) - 1))) * a.c.kv_heads + h;
    const int lane = threadIdx.x & (LANES - 1), d = 4 * lane;
    if (a.acc && lane == 0) a.acc[(static_cast<long long>(b) * a.c.kv_heads + h) * a.acc_cap + p] = 0.0f;
    const int width[2] = {a.c.qk, a.c.vd};
    float x[2][4];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        if (d < width[z]) {
            load_four(x[z], a.x[z], a.type,
                       static_cast<long long>(b) * a.stream[z] + static_cast<long long>(i) * a.row[z] +
                           static_cast<long long>(h) * width[z] + d,
                       vec >> z & 1);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[z][e] = 0.0f;
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        unsigned char *dst = z ? a.c.v : a.c.k;
        const long long at = to * width[z] + d;
        const bool live = d < width[z];
        if constexpr (TYPE == 3) {
            // QuantizeRow (int8.go:36-55) over the head's values
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) m = go_max(m, fabsf(x[z][e]));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) m = go_max(m, __shfl_xor(m, o));
            const float sc = m > 0.0f ? m / 127.0f : 1.0f;
            if (live) {
                uint32_t q = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    q |= (static_cast<uint32_t>(go_int8_code(rintf(x[z][e] / sc))) & 255u) << (8 * e);
                *reinterpret_cast<uint32_t *>(dst + at) = q;
            }
            if (lane == 0) (z ? a.c.vs : a.c.ks)[to] = sc;
        } else if (live) {
            if constexpr (TYPE == 0) {
                reinterpret_cast<float4 *>(dst)[at >> 2] = make_float4(x[z][0], x[z][1], x[z][2], x[z][3]);
            } else {
                uint32_t w[2];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint16_t v = TYPE == 1 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[z][e]))
                                                 : __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[z][e]));
                    w[e / 2] = e & 1 ? w[e / 2] | static_cast<uint32_t>(v) << 16 : v;
                }
                reinterpret_cast<uint2 *>(dst)[at >> 2] = make_uint2(w[0], w[1]);
            }
        }
    }
}

template <int TYPE, int LANES>
hipError_t launch_append_lanes(const PagedAppendArgs &a, int vec, hipStream_t s) {
    const long long units = static_cast<long long>(a.batch) * a.t * a.c.kv_heads;  // below 2^32 / 128
    const long long blocks = (units * LANES + 255) / 256;
    hipLaunchKernelGGL((paged_append_kernel<TYPE, LANES>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a,
                       static_cast<unsigned>(units), vec);
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

constexpr int kSelThreads = 1024;  // at most
constexpr long long kCopyPieces = 1 << 12;  // a list's pieces of 16 bytes that one workgroup copies

// A weight's place in the order of weights: larger is kept sooner. Held rows
// (the first sink, the last recent) come before every weight; -0 is 0; a NaN
// is the least.
__device__ __forceinline__ uint32_t weight_key(float w, bool held) {
    const uint32_t u = __float_as_uint(w + 0.0f), s = static_cast<uint32_t>(static_cast<int32_t>(u) >> 31);
    const uint32_t k = u ^ (s | 0x80000000u);
    return held ? 0xffffffffu : w != w ? 0 : k;
}

template <int H>
__device__ __forceinline__ int add_lane(int c) {
    return c + __builtin_bit_cast(int, xor_lane<H>(__builtin_bit_cast(float, c)));
}
__device__ __forceinline__ int wave_sum(int c) {
    return add_lane<32>(add_lane<16>(add_lane<8>(add_lane<4>(add_lane<2>(add_lane<1>(c))))));
}

using words4 = uint32_t __attribute__((ext_vector_type(4)));

// Where a kept row j of stream b, key head h is, and where row i of its new
// cache; false where that is in no page. Bad source pages read page 0.
__device__ __forceinline__ bool kept_place(const EvictArgs &a, int b, int h, int i, int j, long long &from, long long &to) {
    const int mask = (1 << a.c.shift) - 1;
    int sp = j >= 0 ? a.c.pages[static_cast<long long>(b) * a.c.page_stride + (j >> a.c.shift)] : 0;
    const int dp = j >= 0 ? a.dst_pages[static_cast<long long>(b) * a.dst_stride + (i >> a.c.shift)] : -1;
    if (sp < 0 || sp >= a.c.pool_pages) sp = 0;
    from = ((static_cast<long long>(sp) << a.c.shift) + (j & mask)) * a.c.kv_heads + h;
    to = ((static_cast<long long>(dp) << a.c.shift) + (i & mask)) * a.c.kv_heads + h;
    return dp >= 0 && dp < a.c.pool_pages;
}

// The copies of one list by the workgroup that chose its rows, kept[i] in
// LDS: four 16-byte pieces of a key row and a value row a thread at a time.
__device__ __forceinline__ void copy_kept(const EvictArgs &a, int b, int h, const int *kept, int count, int kpieces,
                                          int vpieces) {
    constexpr int kAhead = 4;
    const int pieces = max(kpieces, vpieces), total = count * pieces, threads = blockDim.x;
    for (int x0 = threadIdx.x; x0 < total; x0 += kAhead * threads) {
        words4 kx[kAhead], vx[kAhead];
        float ksc[kAhead], vsc[kAhead];
        long long from[kAhead], to[kAhead];
        int p[kAhead];
        bool ok[kAhead];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
            const int x = x0 + z * threads, i = min(x, total - 1) / pieces;
            p[z] = x - i * pieces;
            ok[z] = kept_place(a, b, h, i, kept[i], from[z], to[z]) && x < total;
        }
#pragma unroll
        for (int z = 0; z < kAhead; ++z)
            if (ok[z]) {
                if (p[z] < kpieces) kx[z] = reinterpret_cast<const words4 *>(a.c.k)[from[z] * kpieces + p[z]];
                if (p[z] < vpieces) vx[z] = reinterpret_cast<const words4 *>(a.c.v)[from[z] * vpieces + p[z]];
                if (a.c.type == 3 && p[z] == 0) {
                    ksc[z] = a.c.ks[from[z]];
                    vsc[z] = a.c.vs[from[z]];
                }
            }
#pragma unroll
        for (int z = 0; z < kAhead; ++z)
            if (ok[z]) {
                if (p[z] < kpieces) __builtin_nontemporal_store(kx[z], reinterpret_cast<words4 *>(a.c.k) + to[z] * kpieces + p[z]);
                if (p[z] < vpieces) __builtin_nontemporal_store(vx[z], reinterpret_cast<words4 *>(a.c.v) + to[z] * vpieces + p[z]);
                if (a.c.type == 3 && p[z] == 0) {
                    a.c.ks[to[z]] = ksc[z];
                    a.c.vs[to[z]] = vsc[z];
                }
            }
    }
}

// The kept rows of one (stream, key head). Row k of a thread is row
// (wavefront * per + k) * 64 + lane, its key in a register (V = 0: read
// each time, for lists past 32,768). The keep-th largest key is built from its
// highest bits down: bits stay set if at least `keep` keys reach the value
// with them (a histogram's atomics would meet in the few exponents that weights
// have: 30 us for 448 rows), until exactly `keep` do.
// Two bits a turn as long as three counts of a wavefront fit one word (eight
// rows a thread, 8192 rows), then one. To keep 2048 rows of 128 bfloat16 values,
// one list and 32 of them, both launches: of 8192 rows 17.9 and 20.6 us, of
// 20,000 26.7 and 37.3, of 32,768 31.8 and 39.4; of 65,000, whose keys are read
// again each turn, 155 and 300.
// Then one pass in row order writes the rows above the key, and the lowest of
// those equal to it. Integer counts throughout: the same rows in every run.
// COPY: the workgroup also copies them, and a stream's first one writes its
// new length (which then is not where the others read the old one).
template <int V, bool COPY>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a, int kpieces, int vpieces) {
    extern __shared__ int kept_sh[];  // COPY: the kept rows
    __shared__ int count_sh[32][3];  // a turn's counts over the wavefronts
    __shared__ int wave_sh[2][kSelThreads / 64];
    const int tid = threadIdx.x, threads = blockDim.x, wave = tid >> 6, lane = tid & 63;
    const int h = blockIdx.x % a.c.kv_heads, b = blockIdx.x / a.c.kv_heads;
    const int n = a.len[b];
    if (n < 0 || n > a.nk_max) return;
    if (COPY && h == 0 && tid == 0) a.len_out[b] = min(n, a.keep);
    const long long bh = static_cast<long long>(b) * a.c.kv_heads + h;
    const float *w = a.acc + bh * a.acc_cap;
    int32_t *kept = a.kept + bh * a.keep;
    float *out = a.acc_out + bh * a.acc_out_cap;
    for (int i = min(n, a.keep) + tid; i < a.keep; i += threads) kept[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += threads) {
            kept[i] = i;
            out[i] = w[i];
            if (COPY) kept_sh[i] = i;
        }
        if (COPY) {
            __syncthreads();
            copy_kept(a, b, h, kept_sh, n, kpieces, vpieces);
        }
        return;
    }
    if (a.keep == 0) return;
    const int per = V ? V : (n + threads - 1) / threads, row0 = wave * per * 64 + lane;  // row k: row0 + 64 k
    if (tid < 96) (&count_sh[0][0])[tid] = 0;
    if (threads < 96) (&count_sh[0][0])[min(tid + 64, 95)] = 0;
    __syncthreads();
    auto key_at = [&](int j, float x) { return j < n ? weight_key(x, (j < a.sink) | (j >= n - a.recent)) : 0; };
    float weights[V ? V : 1];
    uint32_t keys[V ? V : 1];
    if constexpr (V > 0) {  // all loads in flight before the first is used
#pragma unroll
        for (int k = 0; k < V; ++k) weights[k] = w[min(row0 + 64 * k, n - 1)];
#pragma unroll
        for (int k = 0; k < V; ++k) keys[k] = key_at(row0 + 64 * k, weights[k]);
    }
    auto weight_of = [&](int k) {
        if constexpr (V > 0)
            return weights[k];
        else
            return w[min(row0 + 64 * k, n - 1)];
    };
    auto key_of = [&](int k) {
        if constexpr (V > 0)
            return keys[k];
        else
            return key_at(row0 + 64 * k, weight_of(k));
    };
    // The rows whose key reaches each of three values (above 0): counts of at
    // most 512 a wavefront, ten bits each, so one sum serves all (V <= 8; else
    // one value).
    constexpr int kBits = V > 0 && V <= 8 ? 2 : 1;
    auto reach = [&](const uint32_t (&at)[3], int turn, int (&total)[3]) {
        int c = 0;
        if constexpr (V > 0) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                c += keys[k] >= at[0];
                if constexpr (kBits == 2) c += (keys[k] >= at[1] ? 1 << 10 : 0) + (keys[k] >= at[2] ? 1 << 20 : 0);
            }
        } else {
            for (int k = 0; k < per; ++k) c += key_of(k) >= at[0];
        }
        c = wave_sum(c);
        if (lane < (kBits == 2 ? 3 : 1)) atomicAdd(&count_sh[turn][lane], kBits == 2 ? (c >> (10 * lane)) & 1023 : c);
        __syncthreads();
        total[0] = count_sh[turn][0];
        total[1] = count_sh[turn][1];
        total[2] = count_sh[turn][2];
    };
    // thr: the largest value that at least `keep` keys reach; `above` of them
    // pass it. Each turn settles kBits bits of it: the least of the values
    // with them that fewer than `keep` reach stays above it.
    uint32_t thr = 0;
    int above = 0;
    for (int bit = 32 - kBits; bit >= 0; bit -= kBits) {
        const uint32_t at[3] = {thr | (1u << bit), thr | (2u << bit), thr | (3u << bit)};
        int c[3];
        reach(at, bit / kBits, c);
        uint32_t next = thr;
        bool done = false;
#pragma unroll
        for (int z = 0; z < (kBits == 2 ? 3 : 1); ++z) {
            if (done || c[z] < a.keep) {
                if (!done) {
                    above = c[z];
                    done = true;
                }
                continue;
            }
            next = at[z];
            if (c[z] == a.keep) {  // every key that reaches it, and no other
                next = at[z] - 1;
                above = c[z];
                bit = 0;
                done = true;
            }
        }
        thr = next;
    }
    const int need = a.keep - above;  // of the rows that equal the key, the first
    int ups = 0, eqs = 0;
    auto is_equal = [&](int k) { return row0 + 64 * k < n && key_of(k) == thr; };
#pragma unroll(V ? V : 1)
    for (int k = 0; k < (V ? V : per); ++k) {
        ups += __popcll(__ballot(key_of(k) > thr));
        eqs += __popcll(__ballot(is_equal(k)));
    }
    if (lane == 0) wave_sh[0][wave] = ups, wave_sh[1][wave] = eqs;
    __syncthreads();
    int base = 0, eq_base = 0;  // rows above the key, and equal to it, before this wavefront's row k
    for (int i = 0; i < wave; ++i) base += wave_sh[0][i], eq_base += wave_sh[1][i];
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll(V ? V : 1)
    for (int k = 0; k < (V ? V : per); ++k) {
        const bool up_k = key_of(k) > thr, eq_k = is_equal(k);
        const unsigned long long up = __ballot(up_k), eq = __ballot(eq_k);
        const int e = eq_base + __popcll(eq & below);
        if (up_k || (eq_k && e < need)) {
            const int at = base + __popcll(up & below) + min(e, need);
            kept[at] = row0 + 64 * k;
            if (COPY) kept_sh[at] = row0 + 64 * k;
            out[at] = weight_of(k);
        }
        base += __popcll(up);
        eq_base += __popcll(eq);
    }
    if (COPY) {
        __syncthreads();
        copy_kept(a, b, h, kept_sh, a.keep, kpieces, vpieces);
    }
}

// The kept rows copied: a thread takes 16 bytes of a head's key row and the
// same piece of its value row, of two rows half the budget apart (each
// destination row is written whole by its neighbours): four loads in flight
// behind one chain of row, page and pool. The stores go past the L2 to memory at once, not at the
// launch's end, when the L2s give up their dirty lines (16 streams of up to 8192
// rows to 2048, 8 heads of 128, 237 MB read and written: both launches 57.7 ->
// 52.2 us, this one 44 to 46, 5.2 TB/s, under the profiler; the appends and the
// attention's narrower stores gain nothing by it or lose). The scales of int8
// rows ride with the first piece.
// Also the streams' new lengths.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a, int kpieces, int vpieces, int half_rows,
                                                         long long total) {
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (id < a.batch) {
        const int n = a.len[id];
        if (n >= 0 && n <= a.nk_max) a.len_out[id] = min(n, a.keep);
    }
    if (id >= total) return;
    const int pieces = max(kpieces, vpieces), per_row = pieces * a.c.kv_heads;
    const long long bi = id / per_row;
    const int x = static_cast<int>(id - bi * per_row);
    const int h = x / pieces, p = x - h * pieces;
    const int b = static_cast<int>(bi / half_rows), i0 = static_cast<int>(bi - static_cast<long long>(b) * half_rows);
    const int n = a.len[b];  // or already its new value: in [0, nk_max] both or neither
    if (n < 0 || n > a.nk_max) return;
    const int32_t *kept = a.kept + (static_cast<long long>(b) * a.c.kv_heads + h) * a.keep;
    words4 kx[2], vx[2];
    float ksc[2], vsc[2];
    long long to[2];
    bool ok[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int i = i0 + z * half_rows;
        const int j = i < a.keep ? kept[i] : -1;
        long long from;
        ok[z] = kept_place(a, b, h, i, j, from, to[z]);
        if (ok[z]) {
            if (p < kpieces) kx[z] = reinterpret_cast<const words4 *>(a.c.k)[from * kpieces + p];
            if (p < vpieces) vx[z] = reinterpret_cast<const words4 *>(a.c.v)[from * vpieces + p];
            if (a.c.type == 3 && p == 0) {
                ksc[z] = a.c.ks[from];
                vsc[z] = a.c.vs[from];
            }
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
        if (ok[z]) {
            if (p < kpieces) __builtin_nontemporal_store(kx[z], reinterpret_cast<words4 *>(a.c.k) + to[z] * kpieces + p);
            if (p < vpieces) __builtin_nontemporal_store(vx[z], reinterpret_cast<words4 *>(a.c.v) + to[z] * vpieces + p);
            if (a.c.type == 3 && p == 0) {
                a.c.ks[to[z]] = ksc[z];
                a.c.vs[to[z]] = vsc[z];
            }
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
    const int size = a.c.type == 0 ? 4 : a.c.type == 3 ? 1 : 2;
    const int kpieces = a.c.qk * size / 16, vpieces = a.c.vd * size / 16, half_rows = (a.keep + 1) / 2;
    const dim3 grid(static_cast<unsigned>(a.batch) * a.c.kv_heads);
    const bool apart = a.len_out + a.batch <= a.len || a.len + a.batch <= a.len_out;
    // One launch for small lists, a row a thread, unless the new lengths lie
    // over the old ones, which every workgroup of a stream reads (448 rows to
    // 256 of heads of 48 and 64 float16 values, 3584 pieces: 8 streams of 2 heads
    // 12.9 -> 11.5 us; 8 of 8 heads of 64, 4096 pieces: 11.5 -> 10.0; 64 of them: 20.3 -> 15.4; 1000 rows,
    // 8192 pieces: 13.0 -> 12.4; of 2000, 8000 pieces: 13.3 -> 14.6, 32,000: 12.4
    // -> 21.3).
    if (apart && a.nk_max <= kSelThreads && static_cast<long long>(a.keep) * (kpieces + vpieces) <= kCopyPieces) {
        const dim3 block(64 * std::max(1, (a.nk_max + 63) / 64));
        hipLaunchKernelGGL((evict_select_kernel<1, true>), grid, block, sizeof(int) * std::min(a.keep, a.nk_max), s, a, kpieces,
                           vpieces);
        return hipGetLastError();
    }
    // a wavefront for each 512 rows, eight rows a thread (32 past 16 wavefronts)
    const int per = 512;
    const dim3 block(std::min(kSelThreads, 64 * std::max(1, (a.nk_max + per - 1) / per)));
    if (a.nk_max <= 8 * kSelThreads)
        hipLaunchKernelGGL((evict_select_kernel<8, false>), grid, block, 0, s, a, 0, 0);
    else if (a.nk_max <= 32 * kSelThreads)
        hipLaunchKernelGGL((evict_select_kernel<32, false>), grid, block, 0, s, a, 0, 0);
    else
        hipLaunchKernelGGL((evict_select_kernel<0, false>), grid, block, 0, s, a, 0, 0);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const long long total = static_cast<long long>(a.batch) * half_rows * a.c.kv_heads * std::max(kpieces, vpieces);
    const long long blocks = (std::max<long long>(total, a.batch) + 255) / 256;
    hipLaunchKernelGGL(evict_copy_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, kpieces, vpieces,
                       half_rows, total);
    return hipGetLastError();
}

}  // namespace cqhip
