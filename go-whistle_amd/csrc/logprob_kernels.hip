// gfx950 log probabilities, entropy and top alternatives of rows of logits
// (nd_logprobs_dev).
//
// A workgroup holds a part of a row in registers: one pass over the logits.
// With m the part's maximum, l = sum e^(x - m) and t = sum e^(x - m) (x - m):
// log p(x) = (x - m) - log l, entropy = log l - t / l. The parts of a long
// row are joined by a second launch: l and t move to the common maximum M by
// e^(m - M): t' = e^(m - M) (t + (m - M) l).
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {


// A logit's place in the order of alternatives: the larger value, then the
// lower index; a NaN as -inf, -0 as 0. 0 is below every logit.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) {
    const uint32_t u = __float_as_uint((x != x ? -INFINITY : x) + 0.0f);
    const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (static_cast<unsigned long long>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }

// The logit of a key (a NaN as -inf, -0 as 0).
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t u = static_cast<uint32_t>(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}

__device__ __forceinline__ float logit_at(const void *x, int type, long long i) {
    if (type == 0) return static_cast<const float *>(x)[i];
    const uint16_t h = static_cast<const uint16_t *>(x)[i];
    return type == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// x - m of a token, and what follows from the row's m, l, t.
struct RowStats {
    float m, l, t;
};
__device__ __forceinline__ float log_prob(const RowStats &s, float x) {
    if (s.m == -INFINITY) return s.l != s.l ? s.l : -INFINITY;  // a row of -inf (or NaN) alone
    return (x - s.m) - logf(s.l);
}
__device__ __forceinline__ float entropy(const RowStats &s) {
    if (s.m == -INFINITY) return s.l != s.l ? s.l : 0.0f;
    return logf(s.l) - s.t / s.l;
}

// A row's token and its logit, asked for before the row's statistics are known.
struct Given {
    int tok;
    float x;
};
__device__ __forceinline__ Given given_of(const LogprobArgs &a, int r) {
    Given g{-1, 0.0f};
    if (a.lp) {
        g.tok = a.tokens[r];
        if (g.tok >= 0 && g.tok < a.n) g.x = logit_at(a.x, a.type, static_cast<long long>(r) * a.stride + g.tok);
    }
    return g;
}
__device__ __forceinline__ void write_row(const LogprobArgs &a, int r, const RowStats &s, const Given &g) {
    if (a.lp) a.lp[r] = g.tok < 0 ? 0.0f : g.tok >= a.n ? NAN : log_prob(s, g.x);
    if (a.ent) a.ent[r] = entropy(s);
}

// A wavefront's lanes' values in falling order: lane i has the i-th largest
// (a bitonic sort; no NaN).
__device__ __forceinline__ float sort_lanes(float x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int h = size >> 1; h > 0; h >>= 1) {
            const float y = xor_lane(x, h);
            // the lower lane of a pair keeps the larger value in falling runs
            const bool larger = ((lane & h) == 0) == ((lane & size) == 0 || size == 64);
            x = larger ? fmaxf(x, y) : fminf(x, y);
        }
    return x;
}

// A thread's values are pieces of 16 bytes of the row, kThreads pieces
// apart: piece g covers the part's values kPer g - shift and on, shift the
// distance of the part's first value from the 16-byte boundary before it.
// Pieces across an end of the part are read value by value.
//
// The alternatives: the `top`-th largest of 64 lanes' maxima is a bound that
// at least `top` values of the part reach, and the largest such bound of the
// wavefronts leaves few more (about 20 of 16,384 normal values for 10). Those
// are listed in LDS and ranked by counting. A list of more than kLpList (equal
// values, or more than about 40 alternatives of a long row) takes them one after
// the other, two barriers each, and the part is read again for it: its values'
// registers are not held for that. Rows of 16,384 float32 logits, 5 of them and
// 7168: five alternatives 6.3 and 88 us, 40 16.6 and 198, 41 17.0 and 204, 64 308 and
// 5,356; of equal logits five 30 and 453, 64 262 and 3,241. bfloat16: 6.5 and
// 72, 16.5 and 186, 16.8 and 333, 280 and 3,705.
constexpr int kLpList = 512;

template <int TYPE, int WAVES, int VALS>
__global__ __launch_bounds__(64 * WAVES) void logprob_kernel(LogprobArgs a) {
    constexpr int kThreads = 64 * WAVES;
    constexpr int kPer = TYPE == 0 ? 4 : 8;
    constexpr int kLpPieces = VALS / kPer;
    __shared__ float red[4][WAVES];
    __shared__ unsigned long long list[kLpList];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x % a.splits, r = blockIdx.x / a.splits;
    const int i0 = part * a.chunk, count = min(a.chunk, a.n - i0);
    const long long base = static_cast<long long>(r) * a.stride + i0;
    const uintptr_t first = reinterpret_cast<uintptr_t>(a.x) + static_cast<uintptr_t>(base) * (16 / kPer);
    const int shift = static_cast<int>(first & 15) / (16 / kPer);
    // value e of piece k: place kPer (tid + k kThreads) + e - shift of the part
    auto place = [&](int k) { return kPer * (tid + k * kThreads) - shift; };

    Given given{-1, 0.0f};
    if (tid == 0) {
        listed = 0;
        if (a.splits == 1) given = given_of(a, r);
    }
    float v[VALS];
    float m = -INFINITY, most[kLpPieces];
#pragma unroll
    for (int k = 0; k < kLpPieces; ++k) {
        const int i = place(k);
        if (i >= 0 && i + kPer <= count) {
            const uint4 w = *reinterpret_cast<const uint4 *>(first + static_cast<long long>(i) * (16 / kPer));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                if constexpr (TYPE == 0) {
                    v[k * kPer + e] = __uint_as_float(u[e]);
                } else if constexpr (TYPE == 1) {
                    v[k * kPer + e] = static_cast<float>(
                        __builtin_bit_cast(_Float16, static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)))));
                } else {
                    v[k * kPer + e] = __uint_as_float((e & 1) ? (u[e >> 1] & 0xffff0000u) : (u[e >> 1] << 16));
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                v[k * kPer + e] = i + e >= 0 && i + e < count ? logit_at(a.x, TYPE, base + i + e) : -INFINITY;
        }
    }
#pragma unroll
    for (int k = 0; k < kLpPieces; ++k) {
        most[k] = v[k * kPer];
#pragma unroll
        for (int e = 1; e < kPer; ++e) most[k] = fmaxf(most[k], v[k * kPer + e]);
        m = fmaxf(m, most[k]);
    }
    float bound = -INFINITY;
    if (a.top > 0) {
        const float sorted = sort_lanes(m);
        bound = __shfl(sorted, a.top - 1);
        m = __shfl(sorted, 0);
    } else {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, xor_lane(m, o));
    }
    if (lane == 0) red[0][wave] = m, red[3][wave] = bound;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, red[0][w]), bound = fmaxf(bound, red[3][w]);
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, t = 0.0f;
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
        const float d = v[k] - mu;
        const float e = __expf(d);
        l += e;                                // a NaN among the logits is one here
        t = fmaf(e, fmaxf(d, -0x1p100f), t);  // 0 for -inf
    }
    if (a.top > 0) {
#pragma unroll
        for (int k = 0; k < kLpPieces; ++k)
            if (!(most[k] < bound)) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int i = place(k) + e;
                    if (!(v[k * kPer + e] < bound) && i >= 0 && i < count) {
                        const int at = atomicAdd(&listed, 1);
                        if (at < kLpList) list[at] = rank_key(v[k * kPer + e], i);
                    }
                }
            }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        l += xor_lane(l, o);
        t += xor_lane(t, o);
    }
    if (lane == 0) red[1][wave] = l, red[2][wave] = t;
    __syncthreads();
    l = t = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) l += red[1][w], t += red[2][w];
    const RowStats st{m, l, t};
    float *pt = a.part + (static_cast<long long>(r) * a.splits + part) * (4 + 2 * a.top);
    if (tid == 0) {
        if (a.splits == 1) {
            write_row(a, r, st, given);
        } else {
            pt[0] = m;
            pt[1] = l;
            pt[2] = t;
        }
    }
    // alternative q: the value of key `best` (0: the part has fewer)
    auto answer = [&](int q, unsigned long long best) {
        const int i = i0 + key_index(best);
        if (a.splits > 1) {
            pt[4 + 2 * q] = key_value(best);
            pt[5 + 2 * q] = __int_as_float(best ? i : -1);
        } else {
            a.top_idx[static_cast<long long>(r) * a.top + q] = i;
            a.top_lp[static_cast<long long>(r) * a.top + q] = log_prob(st, key_value(best));
        }
    };
    if (a.top == 0) return;
    const int n = listed;
    if (n <= kLpList) {
        for (int x = tid; x < n; x += kThreads) {
            const unsigned long long mine = list[x];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > mine;
            if (rank < a.top) answer(rank, mine);
        }
        for (int x = n + tid; x < a.top; x += kThreads) answer(x, 0);
        return;
    }
    // one after the other: every thread offers its largest below the last one chosen
    unsigned long long mine = 0, last = ~0ull;
    for (int q = 0; q < a.top; ++q) {
        if (q == 0 || mine == last) {
            mine = 0;
            for (int i = tid; i < count; i += kThreads) {
                const unsigned long long key = rank_key(logit_at(a.x, TYPE, base + i), i);
                if (key < last && key > mine) mine = key;
            }
        }
        unsigned long long best = mine;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor(best, o);
            if (other > best) best = other;
        }
        __syncthreads();
        if (lane == 0) list[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            if (list[w] > best) best = list[w];
        last = best;
        if (tid == 0) answer(q, best);
    }
}

// The parts of a row joined: a wavefront a row.
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobArgs a) {
    const int r = blockIdx.x, lane = threadIdx.x;
    const int rec = 4 + 2 * a.top;
    const float *pt = a.part + static_cast<long long>(r) * a.splits * rec;
    const Given given = given_of(a, r);
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, pt[static_cast<long long>(s) * rec]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, t = 0.0f;
    for (int s = lane; s < a.splits; s += 64) {
        const float *p = pt + static_cast<long long>(s) * rec;
        if (p[0] == -INFINITY) {  // nothing above -inf: 0, or NaN
            l += p[1];
            continue;
        }
        const float d = p[0] - mu, f = __expf(d);
        l += f * p[1];
        t += f > 0.0f ? f * (p[2] + d * p[1]) : 0.0f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        l += __shfl_xor(l, o);
        t += __shfl_xor(t, o);
    }
    const RowStats st{m, l, t};
    if (lane == 0) write_row(a, r, st, given);
    // each part's alternatives are in order: a lane walks the parts s = lane, lane + 64, ...
    unsigned long long last = ~0ull;
    for (int q = 0; q < a.top; ++q) {
        unsigned long long best = 0;
        for (int s = lane; s < a.splits; s += 64) {
            const float *p = pt + static_cast<long long>(s) * rec + 4;
            for (int k = 0; k < a.top; ++k) {
                const int i = __float_as_int(p[2 * k + 1]);
                if (i < 0) break;
                const unsigned long long key = rank_key(p[2 * k], i);
                if (key < last) {
                    if (key > best) best = key;
                    break;
                }
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor(best, o);
            if (other > best) best = other;
        }
        last = best;
        if (lane == 0) {
            const int i = key_index(best);
            a.top_idx[static_cast<long long>(r) * a.top + q] = i;
            a.top_lp[static_cast<long long>(r) * a.top + q] = log_prob(st, key_value(best));
        }
    }
}

template <int WAVES, int VALS = 32>
hipError_t launch_rows(const LogprobArgs &a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(static_cast<long long>(a.rows) * a.splits)), block(64 * WAVES);
    switch (a.type) {
        case 0: hipLaunchKernelGGL((logprob_kernel<0, WAVES, VALS>), grid, block, 0, s, a); break;
        case 1: hipLaunchKernelGGL((logprob_kernel<1, WAVES, VALS>), grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL((logprob_kernel<2, WAVES, VALS>), grid, block, 0, s, a); break;
    }
    return hipGetLastError();
}

// Workgroups of `waves` wavefronts of 32 logits a thread; past eight, eight of 64.
hipError_t launch_parts(const LogprobArgs &a, int waves, hipStream_t s) {
    switch (waves) {
        case 1: return launch_rows<1>(a, s);
        case 2: return launch_rows<2>(a, s);
        case 3: return launch_rows<3>(a, s);
        case 4: return launch_rows<4>(a, s);
        case 5: return launch_rows<5>(a, s);
        case 6: return launch_rows<6>(a, s);
        case 7: return launch_rows<7>(a, s);
        case 8: return launch_rows<8>(a, s);
        default: return launch_rows<8, 64>(a, s);
    }
}

}  // namespace

// The fewest wavefronts that hold a row, 32 logits a thread: what a wavefront
// does once (the sort, the sums' exchanges) is then done least (7168 rows,
// five alternatives, float32: 2048 logits 16 us in one, 31 in four, 64 in
// eight; one row of 2048: 4.8, 5.5, 6.0). Up to twice eight's, 64 a thread
// rather than two parts (one row of 32,768 float32 logits 6.5 us against
// 12.1, 2000 rows 45 against 53; but 16 against 22 for the 7168 rows of 2048 and
// 82 against 88 for those of 16,384). Then parts of eight's at most.
void logprob_parts(LogprobArgs &a, bool aligned) {
    const int wave = 64 * 32, slack = aligned ? 0 : 8;  // a piece where rows start inside one
    const int most = 8 * wave - slack;
    a.splits = a.n <= 16 * wave - slack ? 1 : (a.n + most - 1) / most;
    a.chunk = ((a.n + a.splits - 1) / a.splits + 7) / 8 * 8;
    a.waves = (std::min(a.chunk, a.n) + slack + wave - 1) / wave;
}

hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s) {
    const hipError_t e = launch_parts(a, a.waves, s);
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(logprob_join_kernel, dim3(a.rows), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace cqhip
