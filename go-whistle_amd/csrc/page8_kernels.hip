// gfx950 kernels of 8-bit paged caches with one scale a page and key head
// (the append of kv_append_paged_dev), and the read-back of paged caches of
// any type (kv_read_paged_dev).
//
// The values of a (page, head) are scale * code, scale the largest |x| that
// the page has held since it was begun over 127 (int8) or 448 (e4m3), codes the
// nearest to x / scale. Rows that raise the scale of a begun page have the
// codes of the rows before them rounded anew under the new one.
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>
#include <type_traits>

namespace cqhip {
namespace {

constexpr int kHold = 4;  // steps of a unit's new rows kept in registers

template <int TYPE>
constexpr float kMost = TYPE == 3 ? 127.0f : 448.0f;

// Four values of a row, from an array of `type` (vec: its pieces of four are
// aligned to their size), widened.
__device__ __forceinline__ void load_row4(float *x, const void *p, int type, long long at, bool vec) {
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

// Eight of them (vec: their 16-byte pieces are aligned).
__device__ __forceinline__ void load_row8(float *x, const void *p, int type, long long at, bool vec) {
    if (type != 0 && vec) {
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1)));
            x[e] = type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
        }
    } else {
        load_row4(x, p, type, at, vec);
        load_row4(x + 4, p, type, at + 4, vec);
    }
}

// The codes of four quotients; NaN is 0 in int8 and NaN in e4m3.
template <int TYPE>
__device__ __forceinline__ uint32_t four_codes(const float *r) {
    if constexpr (TYPE == 3) {
        uint32_t q = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = rintf(r[e]);
            q |= (static_cast<uint32_t>(y != y ? 0 : static_cast<int>(fminf(fmaxf(y, -127.0f), 127.0f))) & 255u) << (8 * e);
        }
        return q;
    } else {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = r[e] != r[e] ? r[e] : fminf(fmaxf(r[e], -448.0f), 448.0f);
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
    }
}

// The codes of eight values under a scale: of float32(x / scale). FINITE: no
// value is infinite or NaN, none of the quotients is past the type's largest code
// by more than its rounding, and the scale is in [2^-60, 2^60]. Then inv = float32(1
// / scale) gives a quotient within two of its last places, one step r = x - q
// scale, q + r inv (each rounded once) one within one, and a second step the
// rounded quotient itself (Markstein): five operations where the division's are
// ten, with its ranges. 32 prompts of up to 448 rows of 8 heads of 128, bfloat16 to
// e4m3, 44 MB: 21.3 us with the division and four values a lane, 18.8 so; the floor
// is 8.5, and what is left are the waits rows, position -> page, values ->
// scale of two rounds of wavefronts.
template <int TYPE, bool FINITE>
__device__ __forceinline__ uint2 eight_codes(const float *x, float div, float inv) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (FINITE) {
            const float q = x[e] * inv, q1 = fmaf(fmaf(-q, div, x[e]), inv, q);
            y[e] = fmaf(fmaf(-q1, div, x[e]), inv, q1);
        } else {
            y[e] = x[e] / div;
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const float *r = y + 4 * g;
        if constexpr (!FINITE) {
            w[g] = four_codes<TYPE>(r);
        } else if constexpr (TYPE == 3) {
            // two's complement in the low bytes of 1.5 2^23 + the nearest integer
            constexpr float kMagic = 12582912.0f;
            const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(r[1] + kMagic), __float_as_uint(r[0] + kMagic), 0x0c0c0400u);
            const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(r[3] + kMagic), __float_as_uint(r[2] + kMagic), 0x04000c0cu);
            w[g] = ab | cd;
        } else {
            const int v = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
            w[g] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], v, true));
        }
    }
    return make_uint2(w[0], w[1]);
}

template <int TYPE>
__device__ __forceinline__ void four_values(float *x, uint32_t w) {
    if constexpr (TYPE == 3) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int32_t>(w << (24 - 8 * e)) >> 24);
    } else {
        const int v = static_cast<int>(w);
        x[0] = __builtin_amdgcn_cvt_f32_fp8(v, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8(v, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8(v, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8(v, 3);
    }
}

// The unit of work is the keys or the values of one head in one page that a
// stream's rows reach, one to eight wavefronts (four units of one a workgroup): LANES
// lanes hold a row at eight values each. The page's new rows are asked for before the
// page table's answer, read once (kept in registers up to kHold steps, behind
// those read again) for their bound, then written; the rows before them only
// where the bound raises the scale.
template <int TYPE, int LANES>
__global__ __launch_bounds__(512) void page8_append_kernel(PagedAppendArgs a, int pages_each, unsigned units, int waves, int vec) {
    __shared__ uint32_t wave_max[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tid = waves > 1 ? threadIdx.x : lane, threads = 64 * waves;
    unsigned u = waves > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
    if (u >= units) return;
    const int z = static_cast<int>(u & 1);
    u >>= 1;
    const int h = static_cast<int>(u % a.c.kv_heads);
    u /= a.c.kv_heads;
    const int pi = static_cast<int>(u % pages_each), b = static_cast<int>(u / pages_each);
    const int n = a.rows ? a.rows[b] : a.t;
    const long long p0 = a.pos[b];
    if (n <= 0 || n > a.t) return;
    // the stream's rows that the cache takes: [lo, hi)
    const long long lo = max(p0, 0LL), hi = min(p0 + n, static_cast<long long>(a.cap));
    const long long page = (lo >> a.c.shift) + pi, first = page << a.c.shift;
    const long long from = max(lo, first), to = min(hi, first + (1LL << a.c.shift));
    if (from >= to) return;
    const int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + page];
    const int width = z ? a.c.vd : a.c.qk, d = 8 * (tid & (LANES - 1));
    const bool live = d < width;
    const int per = threads / LANES, r0 = tid / LANES;  // rows a step, this thread's first
    const int count = static_cast<int>(to - from), held = static_cast<int>(from - first);
    const long long src = static_cast<long long>(b) * a.stream[z] + (from - p0) * a.row[z] + static_cast<long long>(h) * width + d;
    const bool v8 = vec >> z & 1;
    float x[kHold][8];
#pragma unroll
    for (int s = 0; s < kHold; ++s) {
        const int r = r0 + s * per;
        if (r < count && live) {
            load_row8(x[s], a.x[z], a.type, src + r * a.row[z], v8);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = 0.0f;
        }
    }
    if (pg < 0 || pg >= a.c.pool_pages) return;
    float *scales = z ? a.c.vs : a.c.ks;
    const long long sat = static_cast<long long>(pg) * a.c.kv_heads + h;
    const float had = held > 0 ? scales[sat] : 0.0f;
    // The bound: the largest |x| by its bits, infinities and NaNs above all; where
    // there are any, once more, of the finite values.
    auto largest = [&](auto of) {
        uint32_t m = 0;
#pragma unroll
        for (int s = 0; s < kHold; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, of(x[s][e]));
        for (int r = r0 + kHold * per; r < count; r += per)
            if (live) {
                float y[8];
                load_row8(y, a.x[z], a.type, src + r * a.row[z], v8);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = max(m, of(y[e]));
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, __float_as_uint(xor_lane(__uint_as_float(m), o)));
        if (waves > 1) {
            __syncthreads();  // the last one's readers are done
            if (lane == 0) wave_max[wave] = m;
            __syncthreads();
            for (int w = 0; w < waves; ++w) m = max(m, wave_max[w]);
        }
        return m;
    };
    constexpr uint32_t kInfinite = 0x7f800000u;
    uint32_t m = largest([](float v) { return __float_as_uint(v) & 0x7fffffffu; });
    const bool finite = m < kInfinite;
    if (!finite)
        m = largest([](float v) {
            const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
            return u < kInfinite ? u : 0u;
        });
    const float sc = fmaxf(had, __uint_as_float(m) / kMost<TYPE>), div = sc > 0.0f ? sc : 1.0f, inv = 1.0f / div;
    const bool plain = finite && div >= 0x1p-60f && div <= 0x1p60f;

    unsigned char *pool = z ? a.c.v : a.c.k;
    const long long row_bytes = static_cast<long long>(a.c.kv_heads) * width;
    unsigned char *at = pool + (static_cast<long long>(pg) << a.c.shift) * row_bytes + static_cast<long long>(h) * width + d;
    auto write = [&](auto all_finite) {
        constexpr bool F = decltype(all_finite)::value;
#pragma unroll
        for (int s = 0; s < kHold; ++s) {
            const int r = r0 + s * per;
            if (r < count && live) *reinterpret_cast<uint2 *>(at + (held + r) * row_bytes) = eight_codes<TYPE, F>(x[s], div, inv);
        }
        for (int r = r0 + kHold * per; r < count; r += per)
            if (live) {
                float y[8];
                load_row8(y, a.x[z], a.type, src + r * a.row[z], v8);
                *reinterpret_cast<uint2 *>(at + (held + r) * row_bytes) = eight_codes<TYPE, F>(y, div, inv);
            }
    };
    if (plain)
        write(std::true_type{});
    else
        write(std::false_type{});
    if (sc != had && live)  // (a scale that was not a number included)
        for (int r = r0; r < held; r += per) {
            uint2 *w = reinterpret_cast<uint2 *>(at + r * row_bytes);
            const uint2 old = *w;
            float y[8];
            four_values<TYPE>(y, old.x);
            four_values<TYPE>(y + 4, old.y);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= had;
            *w = eight_codes<TYPE, false>(y, div, inv);
        }
    if (tid == 0) scales[sat] = sc;
    if (a.acc && z == 0)
        for (int r = tid; r < count; r += threads)
            a.acc[(static_cast<long long>(b) * a.c.kv_heads + h) * a.acc_cap + from + r] = 0.0f;
}

template <int TYPE, int LANES>
hipError_t launch_append(const PagedAppendArgs &a, int vec, hipStream_t s) {
    const int rows = 1 << a.c.shift, most = std::min(rows, a.t);
    const int pages_each = static_cast<int>((static_cast<long long>(a.t) + rows - 2) / rows + 1);
    const long long units = 2LL * a.batch * a.c.kv_heads * pages_each;
    // wavefronts until the held steps take a page's new rows
    int waves = 1;
    while (waves < 8 && most * LANES > 64 * waves * kHold) waves *= 2;
    hipLaunchKernelGGL((page8_append_kernel<TYPE, LANES>), dim3(static_cast<unsigned>(waves > 1 ? units : (units + 3) / 4)),
                       dim3(waves > 1 ? 64 * waves : 256), 0, s, a, pages_each, static_cast<unsigned>(units), waves, vec);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_append_type(const PagedAppendArgs &a, int vec, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return launch_append<TYPE, 8>(a, vec, s);
    if (w <= 128) return launch_append<TYPE, 16>(a, vec, s);
    return launch_append<TYPE, 32>(a, vec, s);
}

// ---- read back --------------------------------------------------------------------

// Eight values from element i on to an array of `type` (vec: its 16-byte pieces are aligned).
__device__ __forceinline__ void store_row8(void *p, int type, long long i, const float *x, bool vec) {
    if (type == 0) {
        float *y = static_cast<float *>(p) + i;
        if (vec) {
            reinterpret_cast<float4 *>(y)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4 *>(y)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e];
        }
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t v = type == 1 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[e]))
                                     : __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[e]));
        w[e / 2] = e & 1 ? w[e / 2] | static_cast<uint32_t>(v) << 16 : v;
    }
    uint16_t *y = static_cast<uint16_t *>(p) + i;
    if (vec) {
        *reinterpret_cast<uint4 *>(y) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
    }
}

// As the append of rows: a head's key row and value row are one unit of LANES
// lanes at eight values each, units in (stream, row, head) order.
template <int TYPE, int LANES>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadArgs a, unsigned units, int vec) {
    const unsigned u = (blockIdx.x * 256u + threadIdx.x) / LANES;
    if (u >= units) return;
    const unsigned bi = u / a.c.kv_heads;
    const int h = static_cast<int>(u - bi * a.c.kv_heads);
    const int b = static_cast<int>(bi / a.t), i = static_cast<int>(bi - static_cast<unsigned>(b) * a.t);
    const int n = a.rows ? a.rows[b] : a.t;  // both asked for before either is looked at
    const long long p = static_cast<long long>(a.pos[b]) + i, page = p >> a.c.shift;
    if (n > a.t || i >= n || p < 0 || page >= a.c.page_stride) return;
    const int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + page];
    if (pg < 0 || pg >= a.c.pool_pages) return;
    const long long row = (static_cast<long long>(pg) << a.c.shift) + (p & ((1 << a.c.shift) - 1));
    const int d = 8 * (threadIdx.x & (LANES - 1));
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int width = z ? a.c.vd : a.c.qk;
        if (d >= width) continue;
        const long long from = (row * a.c.kv_heads + h) * width + d;
        const unsigned char *pool = z ? a.c.v : a.c.k;
        float x[8];
        if constexpr (TYPE == 0) {
            load_row4(x, pool, 0, from, true);
            load_row4(x + 4, pool, 0, from + 4, true);
        } else if constexpr (TYPE <= 2) {
            load_row4(x, pool, TYPE, from, true);
            load_row4(x + 4, pool, TYPE, from + 4, true);
        } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(pool + from);
            four_values<TYPE>(x, w.x);
            four_values<TYPE>(x + 4, w.y);
            const float sc = (z ? a.c.vs : a.c.ks)[(row >> a.c.sshift) * a.c.kv_heads + h];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= sc;
        }
        store_row8(a.y[z], a.type,
                   static_cast<long long>(b) * a.stream[z] + static_cast<long long>(i) * a.row[z] +
                       static_cast<long long>(h) * width + d,
                   x, vec >> z & 1);
    }
}

template <int TYPE, int LANES>
hipError_t launch_read(const PagedReadArgs &a, int vec, hipStream_t s) {
    const long long units = static_cast<long long>(a.batch) * a.t * a.c.kv_heads;
    const long long blocks = (units * LANES + 255) / 256;
    hipLaunchKernelGGL((paged_read_kernel<TYPE, LANES>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a,
                       static_cast<unsigned>(units), vec);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_read_type(const PagedReadArgs &a, int vec, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return launch_read<TYPE, 8>(a, vec, s);
    if (w <= 128) return launch_read<TYPE, 16>(a, vec, s);
    return launch_read<TYPE, 32>(a, vec, s);
}

}  // namespace

hipError_t launch_page8_append(const PagedAppendArgs &a, hipStream_t s) {
    int vec = 0;  // the rows' 16-byte pieces are aligned
    const int size = a.type == 0 ? 4 : 2;
    for (int k = 0; k < 2; ++k)
        if ((reinterpret_cast<uintptr_t>(a.x[k]) | (a.stream[k] * size) | (a.row[k] * size)) % 16 == 0) vec |= 1 << k;
    return a.c.type == 4 ? launch_append_type<4>(a, vec, s) : launch_append_type<3>(a, vec, s);
}

hipError_t launch_paged_read(const PagedReadArgs &a, hipStream_t s) {
    int vec = 0;  // the rows' 16-byte pieces are aligned
    const int size = a.type == 0 ? 4 : 2;
    for (int k = 0; k < 2; ++k)
        if ((reinterpret_cast<uintptr_t>(a.y[k]) | (a.stream[k] * size) | (a.row[k] * size)) % 16 == 0) vec |= 1 << k;
    switch (a.c.type) {
        case 0: return launch_read_type<0>(a, vec, s);
        case 1: return launch_read_type<1>(a, vec, s);
        case 2: return launch_read_type<2>(a, vec, s);
        case 4: return launch_read_type<4>(a, vec, s);
        default: return launch_read_type<3>(a, vec, s);  // int8 with scales a row or a page
    }
}

}  // namespace cqhip
