// gfx950 verification of drafted tokens (nd_verify_drafts_dev).
//
// With p = softmax(target / T) and q = softmax(draft / T) of a row, draft d is
// kept while u q(d) < p(d); the token at the first that is not is the least j
// whose running sum of max(p - q, 0) passes u' times their total, behind the
// last draft that of p. A running sum's next value may be as near to the random
// number as their spacing, about 1 / n, so exponentials and sums are float64:
// at float32's 1e-7 one token in some hundred of 16,384 would be another.
//
// Three launches: every row's parts (the maximum, the sum, the first largest),
// each logit read once (verify_stats_kernel); the parts' sums of the sampled
// row's weights (verify_weights_kernel); the part that the random number falls
// into, added up in order (verify_sample_kernel). The last two derive the
// streams' accepted counts from the first's results by themselves. Greedy
// (T = 0) takes the first and the last.
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

constexpr int kVThreads = 256;
constexpr int kVHold = 16;                     // logits a thread
constexpr int kVChunk = kVThreads * kVHold;    // logits a part
constexpr int kVRecord = 3;                    // doubles of a part: maximum, sum, index of the first largest

// exp(x) for x <= 0: 2^k times the series of exp(r) to r^11, |r| <= ln(2) / 2, off by 6e-15; 0 below -708.
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

__device__ __forceinline__ double shfl_xor_f64(double x, int o) { return __shfl_xor(x, o); }

__device__ __forceinline__ int drafted_of(const VerifyArgs &a, int b) {
    return a.drafted ? min(max(a.drafted[b], 0), a.t) : a.t;
}

// Rows of a stream: the target's t + 1, then the draft's t.
__device__ __forceinline__ int stream_rows(const VerifyArgs &a) { return a.draft ? 2 * a.t + 1 : a.t + 1; }
__device__ __forceinline__ const double *record(const VerifyArgs &a, int b, int row, int part) {
    return a.part + ((static_cast<long long>(b) * stream_rows(a) + row) * a.splits + part) * kVRecord;
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
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += shfl_xor_f64(s, o);
    if (lane == 0) ws[wave] = s;
    __syncthreads();
    if (tid == 0) {
        double *r = const_cast<double *>(record(a, b, row, part));
        r[0] = m;
        r[1] = ((ws[0] + ws[1]) + ws[2]) + ws[3];
        r[2] = j0 + first;
    }
}

// A row's maximum, sum (relative to it) and first largest, by one wavefront.
struct RowStat {
    double m, s;
    int first;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &a, int b, int row) {
    const int lane = threadIdx.x & 63;
    const double it = a.inv_temp == 0.0 ? 1.0 : a.inv_temp;
    double m = -INFINITY;
    int first = INT_MAX;
    for (int p = lane; p < a.splits; p += 64) {  // in order: the first of equals stays
        const double *r = record(a, b, row, p);
        if (r[0] > m) {
            m = r[0];
            first = static_cast<int>(r[2]);
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        const double om = shfl_xor_f64(m, o);
        const int of = __shfl_xor(first, o);
        first = om > m ? of : om == m ? min(first, of) : first;
        m = om > m ? om : m;
    }
    double s = 0.0;
    const double base = m == -INFINITY ? 0.0 : m;
    for (int p = lane; p < a.splits; p += 64) {
        const double *r = record(a, b, row, p);
        s += r[1] * exp_down((r[0] - base) * it);
        if (r[1] != r[1]) s = r[1];  // NaN stays, also of a part of -inf
    }
    for (int o = 32; o > 0; o >>= 1) s += shfl_xor_f64(s, o);
    return {base, s, first};
}

// The least of the drafts that is refused, or their number; by the whole
// workgroup. stat: the target row's and the draft row's there.
struct Decision {
    int a, n;
    RowStat p, q;
};
template <int TYPE>
__device__ Decision decide(const VerifyArgs &a, int b, bool write_lp) {
    __shared__ int refused;
    __shared__ RowStat rows[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int n = drafted_of(a, b);
    if (tid == 0) refused = n;
    __syncthreads();
    const double it = a.inv_temp;
    for (int i = wave; i < n; i += waves) {
        const int d = a.drafts[static_cast<long long>(b) * a.t + i];
        const RowStat p = row_stat(a, b, i);
        bool ok = d >= 0 && d < a.n && p.s > 0.0 && p.s < INFINITY;  // p.s: no NaN
        if (ok) {
            const double x = logit<TYPE>(a.target, b * a.target_stream + i * a.target_row + d);
            if (it == 0.0) {
                ok = p.first == d;
            } else {
                const double pd = exp_down((x - p.m) * it) / p.s;
                double qd = 1.0;
                if (a.draft) {
                    const RowStat q = row_stat(a, b, a.t + 1 + i);
                    const double y = logit<TYPE>(a.draft, b * a.draft_stream + i * a.draft_row + d);
                    qd = exp_down((y - q.m) * it) / q.s;
                }
                ok = static_cast<double>(a.u[static_cast<long long>(b) * a.t + i]) * qd < pd;
            }
        }
        if (lane == 0 && !ok) atomicMin(&refused, i);
    }
    __syncthreads();
    const int at = refused;
    if (wave == 0) {
        const RowStat p = row_stat(a, b, at);
        if (lane == 0) rows[0] = p;
    }
    if (wave == waves - 1) {
        const RowStat q = a.draft && at < n ? row_stat(a, b, a.t + 1 + at) : RowStat{0.0, 1.0, 0};
        if (lane == 0) rows[1] = q;
    }
    if (write_lp && a.lp)
        for (int i = wave; i < at; i += waves) {
            const RowStat p = row_stat(a, b, i);
            const int d = a.drafts[static_cast<long long>(b) * a.t + i];
            const double x = logit<TYPE>(a.target, b * a.target_stream + i * a.target_row + d);
            if (lane == 0)
                a.lp[static_cast<long long>(b) * (a.t + 1) + i] =
                    static_cast<float>((x - p.m) * (it == 0.0 ? 1.0 : it) - log(p.s));
        }
    __syncthreads();
    return {at, n, rows[0], rows[1]};
}

// The weight of token j: of the residual, and of p alone.
template <int TYPE>
__device__ __forceinline__ void weights(const VerifyArgs &a, const Decision &c, int b, int j, double &w, double &p) {
    const double x = logit<TYPE>(a.target, b * a.target_stream + c.a * a.target_row + j);
    p = exp_down((x - c.p.m) * a.inv_temp) / c.p.s;
    w = p;
    if (c.a < c.n) {
        if (a.draft) {
            const double y = logit<TYPE>(a.draft, b * a.draft_stream + c.a * a.draft_row + j);
            w = p - exp_down((y - c.q.m) * a.inv_temp) / c.q.s;
            w = w < 0.0 ? 0.0 : w;  // NaN stays
        } else if (a.drafts[static_cast<long long>(b) * a.t + c.a] == j) {
            w = 0.0;
        }
    }
}

__device__ __forceinline__ double *weight_sums(const VerifyArgs &a, int b, int part) {
    return a.part + static_cast<long long>(a.batch) * stream_rows(a) * a.splits * kVRecord +
           (static_cast<long long>(b) * a.splits + part) * 2;
}

template <int TYPE>
__global__ __launch_bounds__(kVThreads) void verify_weights_kernel(VerifyArgs a) {
    __shared__ double ws[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x % a.splits, b = blockIdx.x / a.splits;
    const Decision c = decide<TYPE>(a, b, false);
    const int j0 = part * a.chunk, count = min(a.chunk, a.n - j0);
    double w = 0.0, p = 0.0;
#pragma unroll 4
    for (int j = tid; j < count; j += kVThreads) {
        double wj, pj;
        weights<TYPE>(a, c, b, j0 + j, wj, pj);
        w += wj;
        p += pj;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        w += shfl_xor_f64(w, o);
        p += shfl_xor_f64(p, o);
    }
    if (lane == 0) {
        ws[0][wave] = w;
        ws[1][wave] = p;
    }
    __syncthreads();
    if (tid < 2) weight_sums(a, b, part)[tid] = ((ws[tid][0] + ws[tid][1]) + ws[tid][2]) + ws[tid][3];
}

template <int TYPE>
__global__ __launch_bounds__(kVThreads) void verify_sample_kernel(VerifyArgs a) {
    __shared__ int chosen, from_p, pass_sh, last_sh;
    __shared__ double rest;
    __shared__ double wave_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
    const Decision c = decide<TYPE>(a, b, true);
    int token = -1;
    if (a.inv_temp == 0.0) {
        if (c.p.s > 0.0 && c.p.s < INFINITY) token = c.p.first;
    } else {
        // the part that u' of the total falls into, and how much of it
        if (tid == 0) {
            double total[2] = {0.0, 0.0};
            for (int p = 0; p < a.splits; ++p)
                for (int k = 0; k < 2; ++k) total[k] += weight_sums(a, b, p)[k];
            const int k = total[0] > 0.0 && total[0] < INFINITY ? 0 : 1;
            int part = -1;
            double left = 0.0;
            if (total[k] > 0.0 && total[k] < INFINITY) {
                const double want = static_cast<double>(a.u_next[b]) * total[k];
                double sum = 0.0;
                for (int p = 0; p < a.splits; ++p) {
                    const double w = weight_sums(a, b, p)[k];
                    if (w > 0.0) {
                        part = p;  // the last one of any weight, if none passes
                        left = want - sum;
                        if (sum + w > want) break;
                    }
                    sum += w;
                }
            }
            chosen = part;
            from_p = k;
            rest = left;
            pass_sh = INT_MAX;
            last_sh = -1;
        }
        __syncthreads();
        if (chosen >= 0) {
            // a thread has kVHold tokens side by side
            const int j0 = chosen * a.chunk, count = min(a.chunk, a.n - j0);
            double w[kVHold], mine = 0.0;
#pragma unroll
            for (int k = 0; k < kVHold; ++k) {
                const int j = tid * kVHold + k;
                double wj = 0.0, pj = 0.0;
                if (j < count) weights<TYPE>(a, c, b, j0 + j, wj, pj);
                w[k] = from_p ? pj : wj;
                mine += w[k];
            }
            double before = mine;  // the running sum up to this thread's last
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double y = __shfl_up(before, o);
                if (lane >= o) before += y;
            }
            if (lane == 63) wave_sum[wave] = before;
            __syncthreads();
            before -= mine;
            for (int v = 0; v < wave; ++v) before += wave_sum[v];
            // the first token whose sum passes, else the last one of any weight
            int pass = INT_MAX, last = -1;
            double sum = before;
#pragma unroll
            for (int k = 0; k < kVHold; ++k) {
                sum += w[k];
                if (w[k] > 0.0) {
                    last = j0 + tid * kVHold + k;
                    if (pass == INT_MAX && sum > rest) pass = last;
                }
            }
            if (pass != INT_MAX) atomicMin(&pass_sh, pass);
            if (last >= 0) atomicMax(&last_sh, last);
            __syncthreads();
            token = pass_sh != INT_MAX ? pass_sh : last_sh;
        }
    }
    const long long row = static_cast<long long>(b) * (a.t + 1);
    for (int i = tid; i <= a.t; i += kVThreads) {
        a.tokens[row + i] = i < c.a ? a.drafts[static_cast<long long>(b) * a.t + i] : i == c.a ? token : -1;
        if (a.lp && i >= c.a) {
            float lp = 0.0f;
            if (i == c.a && token >= 0) {
                const double x = logit<TYPE>(a.target, b * a.target_stream + c.a * a.target_row + token);
                lp = static_cast<float>((x - c.p.m) * (a.inv_temp == 0.0 ? 1.0 : a.inv_temp) - log(c.p.s));
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
    if (a.inv_temp != 0.0)
        hipLaunchKernelGGL((verify_weights_kernel<TYPE>), dim3(static_cast<unsigned>(a.batch) * a.splits), dim3(kVThreads), 0, s, a);
    hipLaunchKernelGGL((verify_sample_kernel<TYPE>), dim3(a.batch), dim3(kVThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

size_t verify_parts(VerifyArgs &a, int cus) {
    (void)cus;
    a.chunk = kVChunk;
    a.splits = (a.n + kVChunk - 1) / kVChunk;
    const size_t rows = a.draft ? 2 * static_cast<size_t>(a.t) + 1 : static_cast<size_t>(a.t) + 1;
    return (rows * kVRecord + 2) * a.batch * a.splits * sizeof(double);
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) {
    return a.type == 0 ? launch_type<0>(a, s) : a.type == 1 ? launch_type<1>(a, s) : launch_type<2>(a, s);
}

}  // namespace cqhip
