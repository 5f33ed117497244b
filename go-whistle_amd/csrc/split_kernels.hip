// gfx950 attention of few query rows over long key lists, split over the
// list's length (kv_attend_paged_dev, and nd_cross_attend_dev in float32 or
// of few rows).
//
// Per (stream, key head) the query columns are the heads of the group times
// the query rows. o = sum_j w_j v_j with w = softmax(q.k_j / scale), one pass
// over the keys with a running maximum m and sum l (in log2 units, p_j =
// 2^(l_j - m)): a wavefront takes tiles of 16 or 32 keys, four wavefronts
// share a workgroup's part of the list and are joined in LDS; the parts of
// one list are joined by a second launch.
//
// Both products run on v_mfma_f32_16x16x4_f32 with everything widened to
// float32, which keeps float32's accuracy for every type and needs no
// shuffle:
//   S = K q^T: A row r (lane % 16) is key r, the contraction index c (lane /
//     16) a 16-byte piece of the key row, so a lane's global load is its
//     operand; element e of the piece goes to the e-th MFMA, whose B operand
//     is the query's same element. S has key 4c + i in register i of lane
//     (column, c).
//   O = V^T P: the register P_i is the B operand as it lies (contraction
//     index c is key 4c + i), and A is a lane's piece of value row 4c + i,
//     elements e of 16 lanes the rows of the e-th MFMA. m and l belong to
//     the lane's column throughout.
#include "cq_internal.hpp"
#include "cq_device.hpp"

#include <algorithm>

namespace cqhip {
namespace {

using f32x4 = float __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kCols = 16;

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
    } else {
        return static_cast<float>(static_cast<int32_t>(w[e >> 2] << (24 - 8 * (e & 3))) >> 24);
    }
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

// The keys of a stream: two spans of row numbers, or the first n rows of a memory.
struct KeyList {
    int lo0, n0, lo1, n;
    bool ok;
    __device__ int row(int j) const { return j < n0 ? lo0 + j : lo1 + (j - n0); }
};

__device__ __forceinline__ KeyList key_list(const SplitArgs &a, int b, int mem) {
    KeyList l{0, 0, 0, 0, true};
    if (a.spans) {
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

__device__ __forceinline__ int q_rows(const SplitArgs &a, int b) { return a.q_len ? min(max(a.q_len[b], 0), a.t) : a.t; }

// Keys a part of the list takes: whole tiles of 32 keys a wavefront, equal over the parts.
__device__ __forceinline__ int part_keys(int n, int splits) {
    constexpr int unit = 32 * kWaves;
    const int units = (n + unit - 1) / unit;
    return (units + splits - 1) / splits * unit;
}

// TYPE: the cache's type; D: widths up to D (64, 128, 256).
template <int TYPE, int D>
__global__ __launch_bounds__(64 * kWaves) void attend_split_kernel(SplitArgs a, int col_tiles) {
    constexpr int kSize = TYPE == 0 ? 4 : TYPE == 3 ? 1 : 2;
    constexpr int kPer = 16 / kSize;          // elements of a 16-byte piece of a key row
    constexpr int kPieces = D / (4 * kPer);   // pieces of a key row a lane loads
    constexpr int kVals = D / 16;             // elements of a lane's piece of a value row
    constexpr int kVWords = kVals * kSize / 4;
    constexpr int kSub = D * kSize <= 256 ? 2 : 1;  // 16-key steps of a tile
    constexpr int kTile = 16 * kSub;
    extern __shared__ __align__(16) float smem[];
    float *ml_sh = smem;                      // [waves][2][16]
    float *o_sh = smem + kWaves * 2 * kCols;  // [waves][16][D + 4]
    constexpr int kRow = D + 4;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, c = lane >> 4;
    int id = blockIdx.x;
    const int sp = id % a.splits;
    id /= a.splits;
    const int ct = id % col_tiles;
    id /= col_tiles;
    const int h = id % a.c.kv_heads, b = id / a.c.kv_heads;
    const int group = a.heads / a.c.kv_heads;
    const int mem = a.index ? a.index[b] : b;
    const KeyList kl = key_list(a, b, mem);
    if (!kl.ok) return;
    const int cols = q_rows(a, b) * group;
    const int col0 = ct * kCols;
    if (col0 >= cols) return;
    const int col = col0 + r;  // this lane's column: query row col / group, head col % group of the group
    const bool col_ok = col < cols;
    const int per = part_keys(kl.n, a.splits);
    const int j0 = min(sp * per, kl.n), j1 = min(j0 + per, kl.n);

    // The query's pieces, 1/scale and log2(e) folded in.
    float qv[kPieces * kPer];
    {
        const long long qo = static_cast<long long>(b) * a.q_stream +
                             static_cast<long long>(col_ok ? col / group : 0) * a.q_row +
                             static_cast<long long>(h * group + (col_ok ? col % group : 0)) * a.c.qk;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int d0 = (4 * p + c) * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                qv[p * kPer + e] = col_ok && d0 < a.c.qk ? load_value(a.q, a.type, qo + d0 + e) * a.scale_log2 : 0.0f;
        }
    }

    f32x4 o[kVals];
#pragma unroll
    for (int e = 0; e < kVals; ++e) o[e] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    const long long k_base = a.c.pages ? 0 : static_cast<long long>(mem) * a.k_mem;
    const long long v_base = a.c.pages ? 0 : static_cast<long long>(mem) * a.v_mem;
    const unsigned char *kp = a.c.k + k_base + static_cast<long long>(h) * a.k_head;
    const unsigned char *vp = a.c.v + v_base + static_cast<long long>(h) * a.v_head;
    const bool v_ok = r * kVals < a.c.vd;
    const int last = j1 - 1;

    // The pool (or memory) row of the lane's key of tile j (lanes of a tile;
    // keys past the part's last read that one's row).
    auto row_of = [&](int j) {
        const int row = kl.row(min(j + (lane & (kTile - 1)), last));
        if (!a.c.pages) return row;
        int pg = a.c.pages[static_cast<long long>(b) * a.c.page_stride + (row >> a.c.shift)];
        if (pg < 0 || pg >= a.c.pool_pages) pg = 0;
        return (pg << a.c.shift) + (row & ((1 << a.c.shift) - 1));
    };
    auto load_keys = [&](uint32_t (&kw)[kSub][kPieces][4], int rows) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
            const unsigned char *p = kp + static_cast<long long>(__shfl(rows, 16 * s + r)) * a.k_row;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int d0 = (4 * k + c) * kPer;
                if (d0 < a.c.qk)
                    load_words<4>(kw[s][k], p + d0 * kSize);
                else
                    kw[s][k][0] = kw[s][k][1] = kw[s][k][2] = kw[s][k][3] = 0;
            }
        }
    };

    float *lg = a.logits;
    if (lg) lg += ((static_cast<long long>(b) * a.c.kv_heads + h) * group + (col_ok ? col : 0)) * a.nk_max;
    int j = j0 + wave * kTile;
    constexpr int kStep = kWaves * kTile;
    if (j < j1) {
        int rows = row_of(j);
        uint32_t kw[kSub][kPieces][4];
        load_keys(kw, rows);
        for (; j < j1; j += kStep) {
            // this tile's values, the next tile's rows
            uint32_t vw[kSub][4][kVWords];
            float ksc[kSub][4], vsc[kSub][4];
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const long long row = __shfl(rows, 16 * s + 4 * c + i);
                    if (v_ok) {
                        load_words<kVWords>(vw[s][i], vp + row * a.v_row + r * (kVals * kSize));
                    } else {
#pragma unroll
                        for (int k = 0; k < kVWords; ++k) vw[s][i][k] = 0;
                    }
                    if constexpr (TYPE == 3) {
                        ksc[s][i] = a.c.ks[row * a.c.kv_heads + h];
                        vsc[s][i] = a.c.vs[row * a.c.kv_heads + h];
                    }
                }
            const int jn = j + kStep;
            if (jn < j1) rows = row_of(jn);

            f32x4 sc[kSub];
#pragma unroll
            for (int s = 0; s < kSub; ++s) sc[s] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
#pragma unroll
                for (int e = 0; e < kPer; ++e)
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
                        sc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(kw[s][k], e), qv[k * kPer + e],
                                                                     sc[s], 0, 0, 0);
            if (jn < j1) load_keys(kw, rows);

            float mt = m;
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int jj = j + 16 * s + 4 * c + i;
                    float x = sc[s][i];
                    if constexpr (TYPE == 3) x *= ksc[s][i];
                    if (jj < j1) {
                        if (lg && col_ok) lg[kl.row(jj)] = x;
                    } else {
                        x = -INFINITY;
                    }
                    sc[s][i] = x;
                    mt = fmaxf(mt, x);
                }
            mt = fmaxf(mt, xor_lane<16>(mt));
            mt = fmaxf(mt, xor_lane<32>(mt));
            const float mu = mt == -INFINITY ? 0.0f : mt;  // no key above -inf so far: every weight 0
            const float f = exp2f(m - mu);
            m = mt;
            l *= f;
#pragma unroll
            for (int e = 0; e < kVals; ++e) o[e] *= f;
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float p = exp2f(sc[s][i] - mu);
                    l += p;
                    if constexpr (TYPE == 3) p *= vsc[s][i];
#pragma unroll
                    for (int e = 0; e < kVals; ++e)
                        o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(vw[s][i], e), p, o[e], 0, 0, 0);
                }
        }
    }
    l += xor_lane<16>(l);
    l += xor_lane<32>(l);

    // Join the wavefronts.
    if (c == 0) {
        ml_sh[(wave * 2) * kCols + r] = m;
        ml_sh[(wave * 2 + 1) * kCols + r] = l;
    }
    __syncthreads();
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mt = fmaxf(mt, ml_sh[(w * 2) * kCols + r]);
    const float f = exp2f(m - (mt == -INFINITY ? 0.0f : mt));
#pragma unroll
    for (int e = 0; e < kVals; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o_sh[(wave * kCols + r) * kRow + kVals * (4 * c + i) + e] = o[e][i] * f;
    __syncthreads();
    for (int x = tid; x < kCols * a.c.vd; x += 64 * kWaves) {
        const int n = x / a.c.vd, d = x - n * a.c.vd, cn = col0 + n;
        if (cn >= cols) break;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, ml_sh[(w * 2) * kCols + n]);
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            sum += ml_sh[(w * 2 + 1) * kCols + n] * exp2f(ml_sh[(w * 2) * kCols + n] - (mx == -INFINITY ? 0.0f : mx));
            v += o_sh[(w * kCols + n) * kRow + d];
        }
        const int head = h * group + cn % group;
        if (a.part) {
            const long long pi = ((static_cast<long long>(b) * a.t + cn / group) * a.heads + head) * a.splits + sp;
            a.part[pi * a.c.vd + d] = v;
            if (d == 0) {
                a.part_ml[2 * pi] = mx;
                a.part_ml[2 * pi + 1] = sum;
            }
        } else {
            store_value(a.out, a.type,
                        static_cast<long long>(b) * a.out_stream + static_cast<long long>(cn / group) * a.out_row +
                            static_cast<long long>(head) * a.c.vd + d,
                        sum == 0.0f ? 0.0f : v / sum);
        }
    }
}

// The parts of a list joined: one wavefront an output row (stream, query row, head).
__global__ __launch_bounds__(256) void attend_join_kernel(SplitArgs a, long long rows) {
    const int lane = threadIdx.x & 63;
    const long long id = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (id >= rows) return;
    const int head = static_cast<int>(id % a.heads);
    const int i = static_cast<int>(id / a.heads % a.t), b = static_cast<int>(id / a.heads / a.t);
    if (!key_list(a, b, a.index ? a.index[b] : b).ok || i >= q_rows(a, b)) return;
    const float *ml = a.part_ml + 2 * id * a.splits;
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int s = lane; s < a.splits; s += 64) l += ml[2 * s + 1] * exp2f(ml[2 * s] - mu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    const float *p = a.part + id * a.splits * a.c.vd;
    for (int d = lane; d < a.c.vd; d += 64) {
        float v = 0.0f;
        for (int s = 0; s < a.splits; ++s) v = fmaf(p[static_cast<long long>(s) * a.c.vd + d], exp2f(ml[2 * s] - mu), v);
        store_value(a.out, a.type,
                    static_cast<long long>(b) * a.out_stream + static_cast<long long>(i) * a.out_row +
                        static_cast<long long>(head) * a.c.vd + d,
                    l == 0.0f ? 0.0f : v / l);
    }
}

// acc_out = acc + the group's softmax weights, a thread a key: key_blocks
// workgroups of 256 keys for each (stream, key head).
__global__ __launch_bounds__(256) void attend_weights_kernel(SplitArgs a, int key_blocks) {
    extern __shared__ __align__(16) float smem[];  // per group head: maximum, 1 / sum
    const int blk = blockIdx.x % key_blocks, id = blockIdx.x / key_blocks;
    const int h = id % a.c.kv_heads, b = id / a.c.kv_heads;
    const int group = a.heads / a.c.kv_heads;
    const KeyList kl = key_list(a, b, b);
    if (blk * 256 >= kl.n) return;
    const int j = blk * 256 + static_cast<int>(threadIdx.x);
    for (int g = threadIdx.x; g < group; g += 256) {
        const float *ml = a.part_ml + 2 * (static_cast<long long>(b) * a.heads + h * group + g) * a.splits;
        float m = -INFINITY, l = 0.0f;
        for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[2 * s]);
        const float mu = m == -INFINITY ? 0.0f : m;
        for (int s = 0; s < a.splits; ++s) l += ml[2 * s + 1] * exp2f(ml[2 * s] - mu);
        smem[2 * g] = mu;
        smem[2 * g + 1] = l == 0.0f ? 0.0f : 1.0f / l;
    }
    __syncthreads();
    if (j >= kl.n) return;
    const int row = kl.row(j);
    const float *lg = a.logits + (static_cast<long long>(b) * a.c.kv_heads + h) * group * a.nk_max + row;
    float w = 0.0f;
    for (int g = 0; g < group; ++g) w += exp2f(lg[static_cast<long long>(g) * a.nk_max] - smem[2 * g]) * smem[2 * g + 1];
    const long long at = (static_cast<long long>(b) * a.c.kv_heads + h) * a.acc_cap + row;
    a.acc_out[at] = (a.acc ? a.acc[at] : 0.0f) + w;
}

template <int TYPE, int D>
hipError_t launch_split(const SplitArgs &a, int col_tiles, unsigned grid, hipStream_t s) {
    constexpr size_t lds = sizeof(float) * (kWaves * 2 * kCols + kWaves * kCols * (D + 4));
    static std::atomic<unsigned long long> attr{0};
    if (lds > 64 * 1024)
        if (hipError_t e = lds_limit_once(reinterpret_cast<const void *>(&attend_split_kernel<TYPE, D>), lds, attr)) return e;
    hipLaunchKernelGGL((attend_split_kernel<TYPE, D>), dim3(grid), dim3(64 * kWaves), lds, s, a, col_tiles);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch_split_width(const SplitArgs &a, int col_tiles, unsigned grid, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return launch_split<TYPE, 64>(a, col_tiles, grid, s);
    if (w <= 128) return launch_split<TYPE, 128>(a, col_tiles, grid, s);
    return launch_split<TYPE, 256>(a, col_tiles, grid, s);
}

}  // namespace

bool split_widths_ok(int qk, int vd) { return qk > 0 && vd > 0 && qk % 16 == 0 && vd % 16 == 0 && qk <= 256 && vd <= 256; }

hipError_t launch_attend_join(const SplitArgs &a, hipStream_t s) {
    const long long rows = static_cast<long long>(a.batch) * a.t * a.heads;
    hipLaunchKernelGGL(attend_join_kernel, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, s, a, rows);
    return hipGetLastError();
}

hipError_t launch_attend_split(const SplitArgs &a, hipStream_t s) {
    const int group = a.heads / a.c.kv_heads;
    const int col_tiles = (a.t * group + kCols - 1) / kCols;
    const unsigned grid = static_cast<unsigned>(static_cast<long long>(a.batch) * a.c.kv_heads * col_tiles * a.splits);
    hipError_t e = a.c.type == 0   ? launch_split_width<0>(a, col_tiles, grid, s)
                   : a.c.type == 1 ? launch_split_width<1>(a, col_tiles, grid, s)
                   : a.c.type == 2 ? launch_split_width<2>(a, col_tiles, grid, s)
                                   : launch_split_width<3>(a, col_tiles, grid, s);
    if (e != hipSuccess || !a.part) return e;
    if ((e = launch_attend_join(a, s)) != hipSuccess) return e;
    if (a.acc_out) {
        const int blocks = (a.nk_max + 255) / 256;
        hipLaunchKernelGGL(attend_weights_kernel, dim3(static_cast<unsigned>(a.batch) * a.c.kv_heads * blocks),
                           dim3(256), sizeof(float) * 2 * group, s, a, blocks);
    }
    return hipGetLastError();
}

}  // namespace cqhip
