// gfx950 norms of the query and key heads with their rotation in one pass
// (nd_qk_norm_rope_dev): per head y = gain x / sqrt(mean(x^2) + 1e-6)
// (ZCRMSNorm, internal/needle/norm.go:53-109, per head as normRotate,
// attention.go:298-330), then the pairs (i, i + width/2) rotated by the table's
// row (rope.go:69-81).
//
// A head is LANES lanes; a lane has V values of the first half and the V that
// they turn with, of the second. One read and one write of every value, so memory
// bounds it: 32 prompts of up to 448 rows, 16 and 4 heads of 128, bfloat16, from a
// packed product: 18.0 us a launch, 77 MB at 4.3 TB/s; one row of 256 streams, 4.9.
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

template <int TYPE, int V>
__device__ __forceinline__ void load_values(float *x, const void *p, long long at, bool vec) {
    if constexpr (TYPE == 0) {
        const float *s = static_cast<const float *>(p) + at;
        if (vec) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 u = *reinterpret_cast<const float4 *>(s + e);
                x[e] = u.x, x[e + 1] = u.y, x[e + 2] = u.z, x[e + 3] = u.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = s[e];
        }
    } else {
        const uint16_t *s = static_cast<const uint16_t *>(p) + at;
        uint32_t w[V / 2];
        if (vec) {
#pragma unroll
            for (int e = 0; e < V; e += 8) *reinterpret_cast<uint4 *>(w + e / 2) = *reinterpret_cast<const uint4 *>(s + e);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2) w[e / 2] = s[e] | static_cast<uint32_t>(s[e + 1]) << 16;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint16_t h = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
            x[e] = TYPE == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h))
                             : __uint_as_float(static_cast<uint32_t>(h) << 16);
        }
    }
}

template <int TYPE, int V>
__device__ __forceinline__ void store_values(void *p, long long at, const float *x, bool vec) {
    if constexpr (TYPE == 0) {
        float *d = static_cast<float *>(p) + at;
        if (vec) {
#pragma unroll
            for (int e = 0; e < V; e += 4)
                *reinterpret_cast<float4 *>(d + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = x[e];
        }
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint16_t v = TYPE == 1 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[e]))
                                         : __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[e]));
            w[e / 2] = e & 1 ? w[e / 2] | static_cast<uint32_t>(v) << 16 : v;
        }
        uint16_t *d = static_cast<uint16_t *>(p) + at;
        if (vec) {
#pragma unroll
            for (int e = 0; e < V; e += 8)
                *reinterpret_cast<uint4 *>(d + e) = make_uint4(w[e / 2], w[e / 2 + 1], w[e / 2 + 2], w[e / 2 + 3]);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        }
    }
}

// vec: bit 0 queries, 1 keys, 2 and 3 their outputs: 16-byte pieces are aligned.
template <int TYPE, int LANES>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a, unsigned units, int vec) {
    constexpr int V = TYPE == 0 ? 4 : 8;
    const unsigned u = (blockIdx.x * 256u + threadIdx.x) / LANES;
    if (u >= units) return;
    const unsigned all = a.heads[0] + a.heads[1], bi = u / all;
    int h = static_cast<int>(u - bi * all);
    const int z = h >= a.heads[0];
    if (z) h -= a.heads[0];
    const int b = static_cast<int>(bi / a.t), i = static_cast<int>(bi - static_cast<unsigned>(b) * a.t);
    const int n = a.rows ? a.rows[b] : a.t;  // both asked for before either is looked at
    const long long p = a.cos_t ? static_cast<long long>(a.pos[b]) + i : 0;
    if (n > a.t || i >= n) return;
    const int half = a.width / 2, d = V * (threadIdx.x & (LANES - 1));
    const bool live = d < half;
    float x[2][V];
    const long long at = static_cast<long long>(b) * a.x_stream[z] + static_cast<long long>(i) * a.x_row[z] +
                         static_cast<long long>(h) * a.width + d;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (live) {
            load_values<TYPE, V>(x[k], a.x[z], at + k * half, vec >> z & 1);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[k][e] = 0.0f;
        }
    }
    if (a.gain[z]) {
        // float32 values as ZCRMSNorm has them: squares and sums in float64 (the
        // squares exact, the sum's order another), the mean and the quotient
        // rounded as there. 16-bit ones in float32: their own rounding is far above its.
        const float *gain = a.gain[z] + d;
        if constexpr (TYPE == 0) {
            double s = 0.0;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) s = fma(static_cast<double>(x[k][e]), static_cast<double>(x[k][e]), s);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
            const float r = zc_rms(s, 0.0, 0.0, 0.0, a.width);
            if (live) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[k][e] = gain[k * half + e] * x[k][e] / r;
            }
        } else {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) s = fmaf(x[k][e], x[k][e], s);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) s += xor_lane(s, o);
            const float r = 1.0f / sqrtf(s / static_cast<float>(a.width) + 1e-6f);
            if (live) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[k][e] *= gain[k * half + e] * r;
            }
        }
    }
    if (!live) return;
    if (a.cos_t) {
        if (p >= 0 && p < a.positions) {
            const float *c = a.cos_t + p * half + d, *s = a.sin_t + p * half + d;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float y0, y1;
                rope_pair(x[0][e], x[1][e], c[e], s[e], y0, y1);
                x[0][e] = y0;
                x[1][e] = y1;
            }
        }
    }
    const long long to = static_cast<long long>(b) * a.y_stream[z] + static_cast<long long>(i) * a.y_row[z] +
                         static_cast<long long>(h) * a.width + d;
#pragma unroll
    for (int k = 0; k < 2; ++k) store_values<TYPE, V>(a.y[z], to + k * half, x[k], vec >> (2 + z) & 1);
}

template <int TYPE, int LANES>
hipError_t launch_lanes(const NormRopeArgs &a, int vec, hipStream_t s) {
    const long long units = static_cast<long long>(a.batch) * a.t * (a.heads[0] + a.heads[1]);
    const long long blocks = (units * LANES + 255) / 256;
    hipLaunchKernelGGL((norm_rope_kernel<TYPE, LANES>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a,
                       static_cast<unsigned>(units), vec);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_type(const NormRopeArgs &a, int vec, hipStream_t s) {
    const int lanes = (a.width / 2 + (TYPE == 0 ? 3 : 7)) / (TYPE == 0 ? 4 : 8);  // up to 32 of float32, 16 of 16 bits
    if (lanes <= 4) return launch_lanes<TYPE, 4>(a, vec, s);
    if (lanes <= 8) return launch_lanes<TYPE, 8>(a, vec, s);
    if constexpr (TYPE == 0)
        if (lanes > 16) return launch_lanes<TYPE, 32>(a, vec, s);
    return launch_lanes<TYPE, 16>(a, vec, s);
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs &a, hipStream_t s) {
    const int size = a.type == 0 ? 4 : 2;
    int vec = 0;
    // half a head is a whole number of 16-byte pieces: width is a multiple of 16
    for (int z = 0; z < 2; ++z) {
        if (((reinterpret_cast<uintptr_t>(a.x[z]) | (a.x_stream[z] * size) | (a.x_row[z] * size)) & 15) == 0) vec |= 1 << z;
        if (((reinterpret_cast<uintptr_t>(a.y[z]) | (a.y_stream[z] * size) | (a.y_row[z] * size)) & 15) == 0) vec |= 4 << z;
    }
    return a.type == 0 ? launch_type<0>(a, vec, s) : a.type == 1 ? launch_type<1>(a, vec, s) : launch_type<2>(a, vec, s);
}

}  // namespace cqhip
