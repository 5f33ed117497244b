// gfx950 verification of drafted tokens (nd_verify_drafts_dev).
//
// With p = softmax(target / T) and q = softmax(draft / T) of a row, draft d is
// kept while u q(d) < p(d); the token at the first that is not is the least j
// whose running sum of max(p - q, 0) passes u' times their total, behind the
// last draft that of p. A running sum's next value may be as near to the random
// number as their spacing, about 1 / n, so exponentials and sums are float64:
// at float32's 1e-7 one token in some hundred of 16,384 would be another.
//
// Two launches. Every row's parts, each logit read once: the maximum, the sum, the
// first largest (verify_stats_kernel). Then a workgroup for each 1024 tokens of
// the row that is sampled: it derives the stream's accepted count from the first
// launch's results by itself and adds up its tokens' weights; the last one of a
// stream to finish finds the token that the random number falls into, by
// wavefronts of 256 tokens, rows of 64, then one of those (verify_choose_kernel;
// greedy, T = 0, needs one workgroup a stream). Some ten waits for memory and
// exchanges bound it where there are few streams, and the float64 units, as an
// exponential is some 25 of their operations: 4 drafts of one stream of 8199 tokens
// 4.8 and 14.4 us (18.6 with 4096 tokens a workgroup of 1024 threads), 8 of 64 streams of 16,384 17
// and 22 (29 with 16 tokens a thread). The last step as a launch of its own: 13 us beside 8.
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

constexpr int kVThreads = 256;
constexpr int kVHold = 16;                     // logits a thread
constexpr int kVChunk = kVThreads * kVHold;    // logits a part
constexpr int kCThreads = 256;                 // of the second launch
constexpr int kCWaves = kCThreads / 64;
constexpr int kCHold = 4;                      // logits a thread there
constexpr int kCChunk = kCThreads * kCHold;    // logits of its parts
constexpr int kVRecord = 3;                    // doubles of a part: maximum, sum, index of the first largest

// exp(x) for x <= 0: 2^k times Taylor's series of exp(r) to r^11, r = x - k ln(2) with ln(2) in two
// parts (Cody and Waite), |r| <= ln(2) / 2, off by 6e-15; 0 below -708.
__device__ __forceinline__ double exp_down(double x) {
    const double k = rint(x * 1.44269504088896338700e+00);
    double r = fma(-k, 6.93147180369123816490e-01, x);
    r = fma(-k, 1.90821492927058770002e-10, r);
    double y = 1.0 / 39916800.0;
    y = fma(y, r, 1.0 / 3628800.0);
    y = fma(y, r, 1.0 / 362880.0);
    y = fma(y, r, 1.0 / 40320.0);
    y = fma(y, r, 1.0 / 5040.0);
    y = fma(y, r, 1.0 / 720.0);
    y = fma(y, r, 1.0 / 120.0);
    y = fma(y, r, 1.0 / 24.0);
    y = fma(y, r, 1.0 / 6.0);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    return x < -708.0 ? 0.0 : ldexp(y, static_cast<int>(fmax(k, -1100.0)));
}

template <int TYPE>
__device__ __forceinline__ float logit(const void *p, long long i) {
    if constexpr (TYPE == 0) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return TYPE == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// Lane l's value from lane l ^ o; the sum over a wavefront, in every lane; the
// running sum up to each lane. By moves within the vector unit where they reach: a
// float64 through the LDS crossbar is two exchanges of some 120 cycles.
__device__ __forceinline__ double shfl_xor_f64(double x, int o) {
    const long long v = __builtin_bit_cast(long long, x);
    const uint32_t lo = __float_as_uint(xor_lane(__uint_as_float(static_cast<uint32_t>(v)), o));
    const uint32_t hi = __float_as_uint(xor_lane(__uint_as_float(static_cast<uint32_t>(v >> 32)), o));
    return __builtin_bit_cast(double, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
}
__device__ __forceinline__ double lanes_sum(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += shfl_xor_f64(x, o);
    return x;
}
__device__ __forceinline__ double lane_value(double x, int lane) {  // the same lane for all
    const long long v = __builtin_bit_cast(long long, x);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return __builtin_bit_cast(double, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
}
template <int N>
__device__ __forceinline__ double row_below(double x) {  // lane - N's value, 0 before the first of a row of 16
    const long long v = __builtin_bit_cast(long long, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x110 + N, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), 0x110 + N, 0xF, 0xF, true);
    return __builtin_bit_cast(double, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
}
__device__ __forceinline__ double running_sum(double x) {
    x += row_below<1>(x);
    x += row_below<2>(x);
    x += row_below<4>(x);
    x += row_below<8>(x);
    const double r0 = lane_value(x, 15), r1 = lane_value(x, 31), r2 = lane_value(x, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return x + (row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r0 + r1 : r0 + r1 + r2);
}

__device__ __forceinline__ int drafted_of(const VerifyArgs &a, int b) {
    return a.drafted ? min(max(a.drafted[b], 0), a.t) : a.t;
}

// Rows of a stream: the target's t + 1, then the draft's t.
__device__ __forceinline__ int stream_rows(const VerifyArgs &a) { return a.draft ? 2 * a.t + 1 : a.t + 1; }
__device__ __forceinline__ const double *record(const VerifyArgs &a, int b, int row, int part) {
    return a.part + ((static_cast<long long>(b) * stream_rows(a) + row) * a.splits + part) * kVRecord;
}

// The second launch's parts: their sums of weights (kNoSum until they are there; a
// sum is 0 or more, or NaN), and how many of a stream have theirs.
constexpr double kNoSum = -1.0;
__device__ __forceinline__ double *weight_sums(const VerifyArgs &a, int b, int part) {
    return a.part + static_cast<long long>(a.batch) * stream_rows(a) * a.splits * kVRecord +
           (static_cast<long long>(b) * a.choose_parts + part) * 2;
}
__device__ __forceinline__ int *finished(const VerifyArgs &a, int b) {
    return reinterpret_cast<int *>(weight_sums(a, a.batch, 0)) + b;
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kVThreads) void verify_stats_kernel(VerifyArgs a) {
    __shared__ float wm[4];
    __shared__ double ws[4];
    __shared__ int wi[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x % a.splits, id = blockIdx.x / a.splits;
    const int rows = stream_rows(a), b = id / rows, row = id - b * rows;
    const int n = drafted_of(a, b);
    const bool target = row <= a.t;
    if (target ? row > n : row - a.t - 1 >= n) return;
    if (row == 0 && part == 0 && a.inv_temp != 0.0) {
        if (tid == 0) *finished(a, b) = 0;
        for (int i = tid; i < 2 * a.choose_parts; i += kVThreads) weight_sums(a, b, 0)[i] = kNoSum;
    }
    const char *base = static_cast<const char *>(target ? a.target : a.draft) +
                       (TYPE == 0 ? 4 : 2) * (target ? b * a.target_stream + row * a.target_row
                                                     : b * a.draft_stream + (row - a.t - 1) * a.draft_row);
    const int j0 = part * a.chunk, count = min(a.chunk, a.n - j0);

    float x[kVHold];
    // the k-th logit of a thread
    constexpr int kPiece = VEC ? (TYPE == 0 ? 4 : 8) : 1;
    auto place = [&](int k) { return (k / kPiece * kVThreads + tid) * kPiece + k % kPiece; };
#pragma unroll
    for (int k = 0; k < kVHold; k += kPiece) {
        const int j = place(k);
        if (VEC && j + kPiece <= count) {
            const uint4 w = *reinterpret_cast<const uint4 *>(base + (TYPE == 0 ? 4LL : 2LL) * (j0 + j));
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                if constexpr (TYPE == 0) {
                    x[k + e] = __uint_as_float(v[e & 3]);
                } else {
                    const uint16_t h = static_cast<uint16_t>(v[(e / 2) & 3] >> (16 * (e & 1)));
                    x[k + e] = TYPE == 1 ? static_cast<float>(__builtin_bit_cast(_Float16, h))
                                         : __uint_as_float(static_cast<uint32_t>(h) << 16);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) x[k + e] = j + e < count ? logit<TYPE>(base, j0 + j + e) : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVHold; ++k) m = fmaxf(m, x[k]);
    int first = INT_MAX;
    if (a.inv_temp == 0.0) {
#pragma unroll
        for (int k = kVHold - 1; k >= 0; --k)
            if (x[k] == m) first = place(k);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float om = xor_lane(m, o);
        const int of = __shfl_xor(first, o);
        first = om > m ? of : om == m ? min(first, of) : first;
        m = fmaxf(m, om);
    }
    if (lane == 0) {
        wm[wave] = m;
        wi[wave] = first;
    }
    __syncthreads();
    m = wm[0];
    first = wi[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        first = wm[w] > m ? wi[w] : wm[w] == m ? min(first, wi[w]) : first;
        m = fmaxf(m, wm[w]);
    }
    // relative to the part's maximum (of -inf alone 0: every term is 0)
    const double it = a.inv_temp == 0.0 ? 1.0 : a.inv_temp, dm = m == -INFINITY ? 0.0 : static_cast<double>(m);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kVHold; ++k) s += exp_down((static_cast<double>(x[k]) - dm) * it);
    s = lanes_sum(s);
    if (lane == 0) ws[wave] = s;
    __syncthreads();
    if (tid == 0) {
        double *r = const_cast<double *>(record(a, b, row, part));
        r[0] = m;
        r[1] = ((ws[0] + ws[1]) + ws[2]) + ws[3];
        r[2] = static_cast<double>(j0) + min(first, a.n);  // a.n: no logit is a number, or none was looked for
    }
}

// A row's maximum, sum (relative to it) and first largest, from its parts, by
// `lanes` lanes side by side, lane `at` of them.
struct RowStat {
    double m, s;
    int first;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &a, int b, int row, int lanes, int at) {
    const double it = a.inv_temp == 0.0 ? 1.0 : a.inv_temp;
    // the first of the lane's parts stays in registers; in order: the first of equals stays
    const double *r0 = record(a, b, row, min(at, a.splits - 1));
    const double m0 = r0[0], s0 = r0[1];
    double m = at < a.splits ? m0 : -INFINITY;
    int first = at < a.splits ? static_cast<int>(r0[2]) : INT_MAX;
    for (int p = at + lanes; p < a.splits; p += lanes) {
        const double *r = record(a, b, row, p);
        if (r[0] > m) {
            m = r[0];
            first = static_cast<int>(r[2]);
        }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
        const double om = shfl_xor_f64(m, o);
        const int of = __shfl_xor(first, o);
        first = om > m ? of : om == m ? min(first, of) : first;
        m = om > m ? om : m;
    }
    const double base = m == -INFINITY ? 0.0 : m;
    double s = at < a.splits ? s0 * exp_down((m0 - base) * it) : 0.0;
    if (at < a.splits && s0 != s0) s = s0;  // NaN stays, also of a part of -inf
    for (int p = at + lanes; p < a.splits; p += lanes) {
        const double *r = record(a, b, row, p);
        s += r[1] * exp_down((r[0] - base) * it);
        if (r[1] != r[1]) s = r[1];
    }
    for (int o = lanes / 2; o > 0; o >>= 1) s += shfl_xor_f64(s, o);
    return {base, s, first};
}

// The least of the drafts that is refused, or their number, with the target
// row's and the draft row's statistics there.
struct Decision {
    int a, n;
    RowStat p, q;
};
// The decision of a stream by the whole workgroup, a few lanes a row; with write
// the accepted drafts' log probabilities. What no other load has to answer for is asked
// for first: a row's statistics, its draft, then the draft's logits.
template <int TYPE>
__device__ Decision decide(const VerifyArgs &a, int b, bool write) {
    constexpr int kKeep = 64;  // rows whose statistics LDS keeps
    __shared__ int refused;
    __shared__ RowStat stats[2][kKeep];
    __shared__ float lps[kKeep];
    const int tid = threadIdx.x, n = drafted_of(a, b);
    const int lanes = a.splits <= 4 ? 4 : a.splits <= 16 ? 16 : 64, at = tid & (lanes - 1), step = kCThreads / lanes;
    if (tid == 0) refused = n;
    __syncthreads();
    const double it = a.inv_temp;
    for (int i0 = 0; i0 <= n; i0 += step) {  // every lane takes every turn: the rows past the last repeat it
        const int i = min(i0 + tid / lanes, n);
        const bool draft = i < n;
        const long long bi = static_cast<long long>(b) * a.t + min(i, max(a.t - 1, 0));
        const int d = draft ? a.drafts[bi] : -1;
        const float u = draft && it != 0.0 ? a.u[bi] : 0.0f;
        const bool known = draft && d >= 0 && d < a.n;
        const double x = known ? logit<TYPE>(a.target, b * a.target_stream + i * a.target_row + d) : 0.0f;
        const double y = known && a.draft ? logit<TYPE>(a.draft, b * a.draft_stream + i * a.draft_row + d) : 0.0f;
        const RowStat p = row_stat(a, b, i, lanes, at);
        const RowStat q = a.draft && n > 0 ? row_stat(a, b, a.t + 1 + min(i, n - 1), lanes, at) : RowStat{0.0, 1.0, 0};
        bool ok = known && p.s > 0.0 && p.s < INFINITY;  // p.s: no NaN
        if (it == 0.0) {
            ok = ok && p.first == d;
        } else {
            const double pd = exp_down((x - p.m) * it) / p.s, qd = a.draft ? exp_down((y - q.m) * it) / q.s : 1.0;
            ok = ok && static_cast<double>(u) * qd < pd;
        }
        if (at == 0) {
            if (draft && !ok) atomicMin(&refused, i);
            if (i < kKeep) {
                stats[0][i] = p;
                stats[1][i] = q;
                if (write) lps[i] = ok ? static_cast<float>((x - p.m) * (it == 0.0 ? 1.0 : it) - log(p.s)) : 0.0f;
            }
        }
    }
    __syncthreads();
    Decision c;
    c.a = refused;
    c.n = n;
    if (c.a < kKeep) {
        c.p = stats[0][c.a];
        c.q = stats[1][c.a];
    } else {
        c.p = row_stat(a, b, c.a, lanes, at);
        c.q = a.draft && n > 0 ? row_stat(a, b, a.t + 1 + min(c.a, n - 1), lanes, at) : RowStat{0.0, 1.0, 0};
    }
    if (write && a.lp)
        for (int i = tid; i < min(c.a, kKeep); i += kCThreads) a.lp[static_cast<long long>(b) * (a.t + 1) + i] = lps[i];
    if (write && a.lp)
        for (int i0 = kKeep; i0 < c.a; i0 += step) {
            const int i = min(i0 + tid / lanes, c.a - 1);
            const RowStat p = row_stat(a, b, i, lanes, at);
            const double x = logit<TYPE>(a.target, b * a.target_stream + i * a.target_row + a.drafts[static_cast<long long>(b) * a.t + i]);
            if (at == 0)
                a.lp[static_cast<long long>(b) * (a.t + 1) + i] =
                    static_cast<float>((x - p.m) * (it == 0.0 ? 1.0 : it) - log(p.s));
        }
    return c;
}

// The weight of a token: of the residual, and of p alone.
struct Weight {
    double w, p;
};

// How a stream's sampled row gives the weights of the tokens from j0 on.
template <int TYPE>
struct Weights {
    const VerifyArgs &a;
    const Decision &c;
    long long xo, yo;
    double pinv, qinv;
    int dropped, count;
    bool minus_q;
    __device__ Weights(const VerifyArgs &a, const Decision &c, int b, int j0, int count)
        : a(a), c(c), xo(b * a.target_stream + c.a * a.target_row + j0), yo(b * a.draft_stream + c.a * a.draft_row + j0),
          pinv(1.0 / c.p.s), qinv(1.0 / c.q.s),
          dropped(c.a < c.n && !a.draft ? a.drafts[static_cast<long long>(b) * a.t + c.a] - j0 : -1), count(count),
          minus_q(c.a < c.n && a.draft) {}
    __device__ Weight of(int j, float x, float y) const {
        Weight r;
        r.p = exp_down((x - c.p.m) * a.inv_temp) * pinv;
        r.w = r.p;
        if (minus_q) {
            const double d = r.p - exp_down((y - c.q.m) * a.inv_temp) * qinv;
            r.w = d < 0.0 ? 0.0 : d;  // NaN stays
        }
        if (j == dropped) r.w = 0.0;
        if (j >= count) r.w = r.p = 0.0;
        return r;
    }
    __device__ float target(int j) const { return logit<TYPE>(a.target, xo + min(j, count - 1)); }
    __device__ float draft(int j) const { return minus_q ? logit<TYPE>(a.draft, yo + min(j, count - 1)) : 0.0f; }
    __device__ Weight at(int j) const { return of(j, target(j), draft(j)); }
    // The sums over a wavefront's 256 tokens, lane l's from j = first + l on, in every lane.
    __device__ Weight wave_sum(int j) const {
        float x[kCHold], y[kCHold];
#pragma unroll
        for (int k = 0; k < kCHold; ++k) x[k] = target(j + 64 * k);
#pragma unroll
        for (int k = 0; k < kCHold; ++k) y[k] = draft(j + 64 * k);
        Weight r{0.0, 0.0};
#pragma unroll
        for (int k = 0; k < kCHold; ++k) {
            const Weight z = of(j + 64 * k, x[k], y[k]);
            r.w += z.w;
            r.p += z.p;
        }
        return {lanes_sum(r.w), lanes_sum(r.p)};
    }
};

// The first of n sums that passes `rest` with those before it, which are taken
// off rest, or the last one above 0 (-1: none is). Every wavefront for itself, alike.
template <class F>
__device__ __forceinline__ int pick(int n, double &rest, F sum) {
    const int lane = threadIdx.x & 63;
    int at = -1;
    double before = 0.0, left = rest;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const double w = i0 + lane < n ? sum(i0 + lane) : 0.0, run = running_sum(w);
        const unsigned long long any = __ballot(w > 0.0), over = __ballot(w > 0.0 && before + run > rest);
        if (any) {
            const int i = over ? __ffsll(over) - 1 : 63 - __clzll(any);
            at = i0 + i;
            left = rest - (before + lane_value(run - w, i));
            if (over) break;
        }
        before += lane_value(run, 63);
    }
    rest = left;
    return at;
}

template <int TYPE>
__global__ __launch_bounds__(kCThreads) void verify_choose_kernel(VerifyArgs a) {
    __shared__ double waves[2][kCWaves], rows[kCHold];
    __shared__ int last_one;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool greedy = a.inv_temp == 0.0;
    int part = greedy ? 0 : blockIdx.x % a.choose_parts;
    const int b = greedy ? blockIdx.x : blockIdx.x / a.choose_parts;
    const Decision c = decide<TYPE>(a, b, part == 0);
    int token = -1;
    if (greedy) {
        if (c.p.s > 0.0 && c.p.s < INFINITY) token = c.p.first;
    } else {
        auto part_weights = [&]() {
            return Weights<TYPE>(a, c, b, part * kCChunk, min(kCChunk, a.n - part * kCChunk));
        };
        auto wave_sums = [&](const Weights<TYPE> &z) {
            const Weight r = z.wave_sum(wave * 64 * kCHold + lane);
            if (lane == 0) {
                waves[0][wave] = r.w;
                waves[1][wave] = r.p;
            }
            __syncthreads();
        };
        wave_sums(part_weights());
        double total[2];
        for (int k = 0; k < 2; ++k) total[k] = lanes_sum(lane < kCWaves ? waves[k][lane] : 0.0);
        // Another part's sum. Its workgroup has counted itself, so the sum is on its way,
        // whether it or the count was seen first.
        auto part_sum = [&](int i, int k) {
            double x;
            do {
                x = __hip_atomic_load(weight_sums(a, b, i) + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            } while (x == kNoSum);
            return x;
        };
        if (a.choose_parts > 1) {
            // The sums pass by the XCDs' own L2s, on either side, so that none of them
            // has to be written back or emptied for a few values (fences of that kind
            // cost 64 streams 15 us). Nothing orders them and the count: a sum that is not
            // there yet says so.
            if (tid < 2) __hip_atomic_store(weight_sums(a, b, part) + tid, total[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (tid == 0)
                last_one = __hip_atomic_fetch_add(finished(a, b), 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.choose_parts - 1;
            __syncthreads();
            if (!last_one) return;
            for (int k = 0; k < 2; ++k) {
                total[k] = 0.0;
                for (int i = lane; i < a.choose_parts; i += 64) total[k] += part_sum(i, k);
                total[k] = lanes_sum(total[k]);
            }
        }
        const int k = total[0] > 0.0 && total[0] < INFINITY ? 0 : 1;  // of the residual, or of p
        if (total[k] > 0.0 && total[k] < INFINITY) {
            double rest = static_cast<double>(a.u_next[b]) * total[k];
            if (a.choose_parts > 1) {
                part = pick(a.choose_parts, rest, [&](int i) { return part_sum(i, k); });
                __syncthreads();  // the sums of this workgroup's own part are read
                wave_sums(part_weights());
            }
            const Weights<TYPE> z = part_weights();
            const int w0 = max(pick(kCWaves, rest, [&](int i) { return waves[k][i]; }), 0) * 64 * kCHold;
            static_assert(kCWaves == kCHold, "a wavefront a row");
            const Weight some = z.at(w0 + wave * 64 + lane);
            const double row_sum = lanes_sum(k ? some.p : some.w);
            if (lane == 0) rows[wave] = row_sum;
            __syncthreads();
            const int j = w0 + max(pick(kCHold, rest, [&](int i) { return rows[i]; }), 0) * 64;
            const Weight one = z.at(j + lane);
            const double w = k ? one.p : one.w;
            token = part * kCChunk + j + max(pick(64, rest, [&](int) { return w; }), 0);
        }
    }
    const long long row = static_cast<long long>(b) * (a.t + 1);
    for (int i = tid; i <= a.t; i += kCThreads) {
        a.tokens[row + i] = i < c.a ? a.drafts[static_cast<long long>(b) * a.t + i] : i == c.a ? token : -1;
        if (a.lp && i >= c.a) {  // those before are written
            float lp = 0.0f;
            if (i == c.a && token >= 0) {
                const double x = logit<TYPE>(a.target, b * a.target_stream + c.a * a.target_row + token);
                lp = static_cast<float>((x - c.p.m) * (greedy ? 1.0 : a.inv_temp) - log(c.p.s));
            }
            a.lp[row + i] = lp;
        }
    }
    if (tid == 0) a.accepted[b] = c.a;
}

template <int TYPE>
hipError_t launch_type(const VerifyArgs &a, hipStream_t s) {
    const int rows = a.draft ? 2 * a.t + 1 : a.t + 1, size = TYPE == 0 ? 4 : 2;
    const auto aligned = [&](const void *p, long long stream, long long row) {
        return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stream * size) | static_cast<uintptr_t>(row * size)) & 15) == 0;
    };
    const bool vec = aligned(a.target, a.target_stream, a.target_row) && (!a.draft || aligned(a.draft, a.draft_stream, a.draft_row));
    const dim3 grid(static_cast<unsigned>(static_cast<long long>(a.batch) * rows * a.splits));
    if (vec)
        hipLaunchKernelGGL((verify_stats_kernel<TYPE, true>), grid, dim3(kVThreads), 0, s, a);
    else
        hipLaunchKernelGGL((verify_stats_kernel<TYPE, false>), grid, dim3(kVThreads), 0, s, a);
    const long long groups = static_cast<long long>(a.batch) * (a.inv_temp == 0.0 ? 1 : a.choose_parts);
    hipLaunchKernelGGL((verify_choose_kernel<TYPE>), dim3(static_cast<unsigned>(groups)), dim3(kCThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

size_t verify_parts(VerifyArgs &a) {
    a.chunk = kVChunk;
    a.splits = (a.n + kVChunk - 1) / kVChunk;
    a.choose_parts = (a.n + kCChunk - 1) / kCChunk;
    const size_t rows = a.draft ? 2 * static_cast<size_t>(a.t) + 1 : static_cast<size_t>(a.t) + 1;
    return a.batch * ((rows * kVRecord * a.splits + 2 * static_cast<size_t>(a.choose_parts)) * sizeof(double) + sizeof(int));
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) {
    return a.type == 0 ? launch_type<0>(a, s) : a.type == 1 ? launch_type<1>(a, s) : launch_type<2>(a, s);
}

}  // namespace cqhip
