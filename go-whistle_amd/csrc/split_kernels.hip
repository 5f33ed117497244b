// gfx950 attention of few query rows over long key lists, split over the
// list's length (kv_attend_paged_dev, and nd_cross_attend_dev in float32 or
// of few rows).
//
// Per (stream, key head) the query columns are the heads of the group times
// the query rows. o = sum_j w_j v_j with w = softmax(q.k_j / scale), one pass
// over the keys with a running maximum m and sum l (in log2 units, p_j =
// 2^(l_j - m)): a wavefront takes tiles of 16 or 32 keys, the wavefronts of a
// workgroup share a part of the list and are joined in LDS; the parts of a
// list, where there are few lists and many keys, by a second launch. Weights,
// softmax and sums are float32, whatever the types.
//
// attend_lanes_kernel, one or two columns (of more, two a workgroup where a
// call has little work: split_tile_columns): lane (r, c) = (lane % 16, lane /
// 16) reads pieces c, c + 4, ... of 16 bytes of key row r and of value row r.
// The logit is the four lanes' sum, and a lane keeps the outputs of its
// pieces for its keys: no exchange of the weights, one sum over r at the end.
// The vector units do it: a piece of 16 int8 keys costs 32 operations a
// column there, and 16 matrix instructions whatever the columns.
//
// attend_split_kernel, three to 16 columns a tile: both products on
// v_mfma_f32_16x16x4_f32 with everything widened to float32, without a
// shuffle:
//   S = K q^T: A row r is key r, the contraction index c a 16-byte piece of
//     the key row, so a lane's global load is its operand; element e of the
//     piece goes to the e-th MFMA, whose B operand is the query's same
//     element. S has key 4c + i in register i of lane (column, c). 16-bit keys,
//     and int8 ones widened to bfloat16 (exactly), take v_mfma_f32_16x16x32
//     instead, eight elements at a time: with the query as it is where it has
//     the keys' type, else as the exact sum of three bfloat16 parts (24 bits).
//     The products are exact either way; the eight float32 instructions that
//     one to three of them replace kept the matrix pipe 57% busy (4 streams of
//     65,000 bfloat16 keys 220 -> 212 us). An infinite key times a part of 0 is
//     NaN: logits that are, are computed again in float32.
//   O = V^T P: the register P_i is the B operand as it lies (contraction
//     index c is key 4c + i), and A is a lane's piece of value row 4c + i,
//     elements e of 16 lanes the rows of the e-th MFMA. m and l belong to
//     the lane's column throughout.
#include "split_device.hpp"

#include <algorithm>
#include <type_traits>

namespace cqhip {
namespace {

// TYPE: the cache's type; D: widths up to D (64, 128, 256); COLS: columns a tile.
template <int TYPE, int D, int COLS>
__global__ __launch_bounds__(D <= 128 ? 512 : 256) void attend_lanes_kernel(SplitArgs a, int col_tiles) {
    constexpr int kSize = kValueSize<TYPE>;
    constexpr int kPer = 16 / kSize;         // elements of a piece
    constexpr int kPieces = D / (4 * kPer);  // pieces of a row a lane reads
    constexpr int kSub = D * kSize <= 128 ? 2 : 1;  // 16-key steps of a tile
    constexpr int kTile = 16 * kSub;
    extern __shared__ __align__(16) float smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, c = lane >> 4;
    const Place p = place_of(a, col_tiles, COLS);
    if (!p.ok) return;
    const Joint<COLS, D> jt(smem, waves);
    const int col0 = p.ct * COLS, nc = min(COLS, p.cols - col0);

    float q[COLS][kPieces * kPer], o[COLS][kPieces * kPer], m[COLS], l[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const long long qo = query_at(a, p, min(col0 + n, p.cols - 1));
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int d0 = (4 * k + c) * kPer;
            if (d0 < a.c.qk) {
                load_query<kPer>(&q[n][k * kPer], a, qo + d0, a.scale_log2);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) q[n][k * kPer + e] = 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < kPieces * kPer; ++e) o[n][e] = 0.0f;
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    const unsigned char *kp = a.c.k + (a.c.pages ? 0 : static_cast<long long>(p.mem) * a.k_mem) + static_cast<long long>(p.h) * a.k_head;
    const unsigned char *vp = a.c.v + (a.c.pages ? 0 : static_cast<long long>(p.mem) * a.v_mem) + static_cast<long long>(p.h) * a.v_head;
    float *lg = a.logits ? a.logits + (static_cast<long long>(p.b) * a.c.kv_heads + p.h) * p.group * a.nk_max : nullptr;

    uint32_t kw[kSub][kPieces][4], vw[kSub][kPieces][4];
    float ks[kSub], vs[kSub];
    int rows[kSub];
    auto rows_of = [&](int j) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) rows[s] = array_row(a, p, min(j + 16 * s + r, p.j1 - 1));
    };
    auto load_rows = [&](uint32_t (&w)[kSub][kPieces][4], const unsigned char *base, long long stride, int width) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
            const unsigned char *at = base + static_cast<long long>(rows[s]) * stride;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int d0 = (4 * k + c) * kPer;
                if (d0 < width)
                    load_words<4>(w[s][k], at + d0 * kSize);
                else
                    w[s][k][0] = w[s][k][1] = w[s][k][2] = w[s][k][3] = 0;
            }
        }
    };
    auto load_scales = [&]() {
        if constexpr (kScaled<TYPE>) {
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
                ks[s] = a.c.ks[scale_at(a, rows[s], p.h)];
                vs[s] = a.c.vs[scale_at(a, rows[s], p.h)];
            }
        }
    };
    const int step = waves * kTile;
    int j = p.j0 + wave * kTile;
    if (j < p.j1) {
        rows_of(j);
        load_rows(kw, kp, a.k_row, a.c.qk);
        load_rows(vw, vp, a.v_row, a.c.vd);
        load_scales();
        if (j + step < p.j1) rows_of(j + step);
        for (; j < p.j1; j += step) {
            const bool more = j + step < p.j1;
            // logits: the four lanes' sums; the keys' registers are then the next tile's
            float x[COLS][kSub];
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int n = 0; n < COLS; ++n) {
                    float d = 0.0f;
#pragma unroll
                    for (int k = 0; k < kPieces; ++k)
#pragma unroll
                        for (int e = 0; e < kPer; ++e) d = fmaf(piece_value<TYPE>(kw[s][k], e), q[n][k * kPer + e], d);
                    d += xor_lane<16>(d);
                    d += xor_lane<32>(d);
                    if constexpr (kScaled<TYPE>) d *= ks[s];
                    x[n][s] = d;
                }
            float vsc[kSub];
#pragma unroll
            for (int s = 0; s < kSub; ++s) vsc[s] = kScaled<TYPE> ? vs[s] : 1.0f;
            if (more) load_rows(kw, kp, a.k_row, a.c.qk);
            // past the last key values of 0, not that key's: a weight of 0 times an infinity
            if (!kFinite<TYPE> && j + kTile > p.j1) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
                    if (j + 16 * s + r >= p.j1) {
#pragma unroll
                        for (int k = 0; k < kPieces; ++k) vw[s][k][0] = vw[s][k][1] = vw[s][k][2] = vw[s][k][3] = 0;
                    }
            }
            float w[COLS][kSub];
#pragma unroll
            for (int n = 0; n < COLS; ++n) {
                float mt = m[n];
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const int jj = j + 16 * s + r;
                    if (jj >= p.j1) {
                        x[n][s] = -INFINITY;
                    } else if (a.acc_out && c == 0 && n < nc) {
                        if (lg)
                            lg[static_cast<long long>(col0 + n) * a.nk_max + p.kl.row(jj)] = x[n][s];
                        else
                            jt.logits[n * a.nk_max + jj] = x[n][s];
                    }
                    mt = fmaxf(mt, x[n][s]);
                }
                mt = row_max(mt);
                const float mu = mt == -INFINITY ? 0.0f : mt;
                const float f = __builtin_amdgcn_exp2f(m[n] - mu);
                m[n] = mt;
                l[n] *= f;
#pragma unroll
                for (int e = 0; e < kPieces * kPer; ++e) o[n][e] *= f;
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const float pw = __builtin_amdgcn_exp2f(x[n][s] - mu);
                    l[n] += pw;
                    w[n][s] = kScaled<TYPE> && j + 16 * s + r >= p.j1 ? 0.0f : pw * vsc[s];
                }
            }
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int k = 0; k < kPieces; ++k)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        const float y = piece_value<TYPE>(vw[s][k], e);
#pragma unroll
                        for (int n = 0; n < COLS; ++n) o[n][k * kPer + e] = fmaf(y, w[n][s], o[n][k * kPer + e]);
                    }
            if (more) {
                load_rows(vw, vp, a.v_row, a.c.vd);
                load_scales();
                if (j + 2 * step < p.j1) rows_of(j + 2 * step);
            }
        }
    }
    // the sums over the keys' lanes, then the wavefronts'
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const float lt = row_sum(l[n]);
        if (lane == 0) {
            jt.ml[(wave * 2) * COLS + n] = m[n];
            jt.ml[(wave * 2 + 1) * COLS + n] = lt;
        }
#pragma unroll
        for (int k = 0; k < kPieces; ++k)
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
                const float *t = &o[n][k * kPer + e];
                const float4 y = make_float4(row_sum(t[0]), row_sum(t[1]), row_sum(t[2]), row_sum(t[3]));
                if (r == 0) *reinterpret_cast<float4 *>(&jt.o[(wave * COLS + n) * jt.kRow + (4 * k + c) * kPer + e]) = y;
            }
    }
    finish<COLS, D>(a, p, jt);
}

// TYPE: the cache's type (codes with a scale a page, 4 and 5, are attend_parts_kernel's);
// D: widths up to D (64, 128, 256); PARTS: 16-bit parts of a query value (0: the
// products of the logits in float32).
template <int TYPE, int D, int PARTS>
__global__ __launch_bounds__(D <= 128 ? 512 : 256) void attend_split_kernel(SplitArgs a, int col_tiles) {
    constexpr int kSize = kValueSize<TYPE>;
    constexpr int kPer = 16 / kSize;          // elements of a 16-byte piece of a key row
    constexpr int kPieces = D / (4 * kPer);   // pieces of a key row a lane loads
    constexpr int kVals = D / 16;             // elements of a lane's piece of a value row
    constexpr int kVWords = kVals * kSize / 4;
    constexpr int kSub = D * kSize <= 256 ? 2 : 1;  // 16-key steps of a tile
    constexpr int kTile = 16 * kSub;
    extern __shared__ __align__(16) float smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, c = lane >> 4;
    const Place p = place_of(a, col_tiles, kCols);
    if (!p.ok) return;
    const Joint<kCols, D> jt(smem, waves);
    const int col = p.ct * kCols + r;  // this lane's column: query row col / group, head col % group of the group
    const bool col_ok = col < p.cols;

    // The query's pieces: in float32 with 1/scale and log2(e) folded in, or in
    // 16-bit parts of eight.
    constexpr int kEights = PARTS ? kPer / 8 : 1;
    float qv[PARTS ? 1 : kPieces * kPer];
    uint32_t qp[PARTS ? PARTS : 1][kPieces][kEights][4];
    {
        const long long qo = query_at(a, p, col_ok ? col : 0);
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int d0 = (4 * k + c) * kPer;
            float x[kPer];
            if (col_ok && d0 < a.c.qk) {
                load_query<kPer>(x, a, qo + d0, PARTS ? 1.0f : a.scale_log2);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) x[e] = 0.0f;
            }
            if constexpr (PARTS == 0) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) qv[k * kPer + e] = x[e];
            } else if constexpr (TYPE == 1) {  // a float16 query
#pragma unroll
                for (int e = 0; e < kPer; e += 2)
                    qp[0][k][e / 8][e / 2 % 4] =
                        __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[e])) |
                        static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x[e + 1]))) << 16;
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) x[e] = __builtin_canonicalizef(x[e]);  // a NaN's mark in the upper half
#pragma unroll
                for (int z = 0; z < PARTS; ++z)
#pragma unroll
                    for (int e = 0; e < kPer; e += 2) {
                        qp[z][k][e / 8][e / 2 % 4] = upper_pair(x[e], x[e + 1]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {  // what the part leaves: nothing of an infinity
                            const float part = __uint_as_float(__float_as_uint(x[e + i]) & 0xffff0000u);
                            x[e + i] = fabsf(part) < INFINITY ? x[e + i] - part : 0.0f;
                        }
                    }
            }
        }
    }

    f32x4 o[kVals];
#pragma unroll
    for (int e = 0; e < kVals; ++e) o[e] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    const unsigned char *kp = a.c.k + (a.c.pages ? 0 : static_cast<long long>(p.mem) * a.k_mem) + static_cast<long long>(p.h) * a.k_head;
    const unsigned char *vp = a.c.v + (a.c.pages ? 0 : static_cast<long long>(p.mem) * a.v_mem) + static_cast<long long>(p.h) * a.v_head;
    const bool v_ok = r * kVals < a.c.vd;

    // Row of the lane's key of a tile (its first kTile lanes; keys past the part's last read that one's row).
    auto row_of = [&](int j) { return array_row(a, p, min(j + (lane & (kTile - 1)), p.j1 - 1)); };
    auto load_keys = [&](uint32_t (&kw)[kSub][kPieces][4], int rows) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
            const unsigned char *at = kp + static_cast<long long>(__shfl(rows, 16 * s + r)) * a.k_row;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int d0 = (4 * k + c) * kPer;
                if (d0 < a.c.qk)
                    load_words<4>(kw[s][k], at + d0 * kSize);
                else
                    kw[s][k][0] = kw[s][k][1] = kw[s][k][2] = kw[s][k][3] = 0;
            }
        }
    };

    float *lg = a.logits;
    if (lg) lg += ((static_cast<long long>(p.b) * a.c.kv_heads + p.h) * p.group + (col_ok ? col : 0)) * a.nk_max;
    const int step = waves * kTile;
    int j = p.j0 + wave * kTile;
    if (j < p.j1) {
        int rows = row_of(j);
        uint32_t kw[kSub][kPieces][4];
        load_keys(kw, rows);
        for (; j < p.j1; j += step) {
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
                        ksc[s][i] = a.c.ks[scale_at(a, row, p.h)];
                        vsc[s][i] = a.c.vs[scale_at(a, row, p.h)];
                    }
                }
            const int jn = j + step;
            if (jn < p.j1) rows = row_of(jn);

            f32x4 sc[kSub];
#pragma unroll
            for (int s = 0; s < kSub; ++s) sc[s] = f32x4{0, 0, 0, 0};
            if constexpr (PARTS == 0) {
#pragma unroll
                for (int k = 0; k < kPieces; ++k)
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
#pragma unroll
                        for (int s = 0; s < kSub; ++s)
                            sc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(kw[s][k], e),
                                                                         qv[k * kPer + e], sc[s], 0, 0, 0);
            } else {
#pragma unroll
                for (int k = 0; k < kPieces; ++k)
#pragma unroll
                    for (int e = 0; e < kEights; ++e)
#pragma unroll
                        for (int s = 0; s < kSub; ++s) {
                            uint32_t ka[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z)
                                ka[z] = TYPE == 3 ? upper_pair(piece_value<TYPE>(kw[s][k], 8 * e + 2 * z),
                                                               piece_value<TYPE>(kw[s][k], 8 * e + 2 * z + 1))
                                                  : kw[s][k][z];
#pragma unroll
                            for (int z = 0; z < PARTS; ++z) sc[s] = mfma_16x16x32<TYPE>(ka, qp[z][k][e], sc[s]);
                        }
            }
            // An infinite key times a part of 0 is NaN: such logits again, in float32.
            if constexpr (PARTS == 3 && TYPE != 3) {
                bool nan = false;
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) nan |= sc[s][i] != sc[s][i];
                if (__any(nan)) {
                    f32x4 y[kSub];
#pragma unroll
                    for (int s = 0; s < kSub; ++s) y[s] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < kPieces; ++k)
#pragma unroll
                        for (int e = 0; e < kPer; ++e) {
                            const float q = (piece_value<2>(qp[0][k][e / 8], e & 7) + piece_value<2>(qp[1][k][e / 8], e & 7)) +
                                            piece_value<2>(qp[2][k][e / 8], e & 7);
#pragma unroll
                            for (int s = 0; s < kSub; ++s)
                                y[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(kw[s][k], e), q, y[s], 0, 0, 0);
                        }
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[s][i] = sc[s][i] != sc[s][i] ? y[s][i] : sc[s][i];
                }
            }
            if (jn < p.j1) load_keys(kw, rows);
            // past the last key values of 0, not that key's: a weight of 0 times an infinity
            if (TYPE != 3 && j + kTile > p.j1) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (j + 16 * s + 4 * c + i >= p.j1) {
#pragma unroll
                            for (int k = 0; k < kVWords; ++k) vw[s][i][k] = 0;
                        }
            }

            float mt = m;
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int jj = j + 16 * s + 4 * c + i;
                    float x = sc[s][i];
                    if constexpr (PARTS > 0) x *= a.scale_log2;
                    if constexpr (TYPE == 3) x *= ksc[s][i];
                    if (jj >= p.j1) {
                        x = -INFINITY;
                    } else if (a.acc_out && col_ok) {
                        if (lg)
                            lg[p.kl.row(jj)] = x;
                        else
                            jt.logits[r * a.nk_max + jj] = x;
                    }
                    sc[s][i] = x;
                    mt = fmaxf(mt, x);
                }
            mt = fmaxf(mt, xor_lane<16>(mt));
            mt = fmaxf(mt, xor_lane<32>(mt));
            const float mu = mt == -INFINITY ? 0.0f : mt;  // no key above -inf so far: every weight 0
            const float f = __builtin_amdgcn_exp2f(m - mu);
            m = mt;
            l *= f;
#pragma unroll
            for (int e = 0; e < kVals; ++e) o[e] *= f;
#pragma unroll
            for (int s = 0; s < kSub; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float w = __builtin_amdgcn_exp2f(sc[s][i] - mu);
                    l += w;
                    if constexpr (TYPE == 3) w = j + 16 * s + 4 * c + i >= p.j1 ? 0.0f : w * vsc[s][i];
#pragma unroll
                    for (int e = 0; e < kVals; ++e)
                        o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(vw[s][i], e), w, o[e], 0, 0, 0);
                }
        }
    }
    l += xor_lane<16>(l);
    l += xor_lane<32>(l);
    if (c == 0) {
        jt.ml[(wave * 2) * kCols + r] = m;
        jt.ml[(wave * 2 + 1) * kCols + r] = l;
    }
    if (col_ok) {
#pragma unroll
        for (int e = 0; e < kVals; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) jt.o[(wave * kCols + r) * jt.kRow + kVals * (4 * c + i) + e] = o[e][i];
    }
    finish<kCols, D>(a, p, jt);
}

// The parts of a list joined: a wavefront 128 values of an output row (stream,
// query row, head), two a lane. The parts' statistics and values are asked
// for before the row's spans or length say whether it is written: the three
// are one wait.
__global__ __launch_bounds__(64) void attend_join_kernel(SplitArgs a, int blocks) {
    const int lane = threadIdx.x;
    const int id = blockIdx.x / blocks, d = (blockIdx.x - id * blocks) * 128 + 2 * lane;
    const int bi = id / a.heads, head = id - bi * a.heads;
    const int b = bi / a.t, i = bi - b * a.t;
    // lane s has part s's maximum and sum; up to 64 parts
    const float *ml = a.part_ml + 2LL * id * a.splits;
    const float2 mine = lane < a.splits ? *reinterpret_cast<const float2 *>(ml + 2 * lane) : make_float2(-INFINITY, 0.0f);
    const float *part = a.part + static_cast<long long>(id) * a.splits * a.c.vd + min(d, a.c.vd - 2);
    constexpr int kAhead = 16;
    float2 x[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) x[s] = *reinterpret_cast<const float2 *>(part + min(s, a.splits - 1) * a.c.vd);
    if ((!a.pos && !key_list(a, b, a.index ? a.index[b] : b).ok) || i >= q_rows(a, b)) return;
    float m = mine.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, xor_lane(m, o));
    const float f = __builtin_amdgcn_exp2f(mine.x - (m == -INFINITY ? 0.0f : m));
    float l = mine.y * f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += xor_lane(l, o);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (s < a.splits) {
            const float fs = __shfl(f, s);
            v.x = fmaf(x[s].x, fs, v.x);
            v.y = fmaf(x[s].y, fs, v.y);
        }
    for (int s = kAhead; s < a.splits; ++s) {
        const float2 y = *reinterpret_cast<const float2 *>(part + s * a.c.vd);
        const float fs = __shfl(f, s);
        v.x = fmaf(y.x, fs, v.x);
        v.y = fmaf(y.y, fs, v.y);
    }
    if (d >= a.c.vd) return;
    const long long at = static_cast<long long>(b) * a.out_stream + static_cast<long long>(i) * a.out_row +
                         static_cast<long long>(head) * a.c.vd + d;
    store_value(a.out, a.type, at, v.x * inv);
    store_value(a.out, a.type, at + 1, v.y * inv);
}

// acc_out = acc + the group's softmax weights from the logits in the
// workspace, a thread a key: key_blocks workgroups of 256 keys for each
// (stream, key head).
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
        for (int s = 0; s < a.splits; ++s) l += ml[2 * s + 1] * __builtin_amdgcn_exp2f(ml[2 * s] - mu);
        smem[2 * g] = mu;
        smem[2 * g + 1] = l == 0.0f ? 0.0f : 1.0f / l;
    }
    __syncthreads();
    if (j >= kl.n) return;
    const int row = kl.row(j);
    const float *lg = a.logits + (static_cast<long long>(b) * a.c.kv_heads + h) * group * a.nk_max + row;
    float w = 0.0f;
    for (int g = 0; g < group; ++g)
        w += __builtin_amdgcn_exp2f(lg[static_cast<long long>(g) * a.nk_max] - smem[2 * g]) * smem[2 * g + 1];
    const long long at = (static_cast<long long>(b) * a.c.kv_heads + h) * a.acc_cap + row;
    a.acc_out[at] = (a.acc ? a.acc[at] : 0.0f) + w;
}

template <int TYPE, int D, int PARTS>
hipError_t launch_columns(const SplitArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> attr{0};
    return launch_with(&attend_split_kernel<TYPE, D, PARTS>, a, kCols, joint_lds<kCols, D>(a, a.waves), attr, s);
}

template <int TYPE, int D>
hipError_t launch_split(const SplitArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> one{0}, two{0};
    const int tile = a.tile;
    if (tile == 1)
        return launch_with(&attend_lanes_kernel<TYPE, D, 1>, a, 1, joint_lds<1, D>(a, a.waves), one, s);
    if (tile == 2)
        return launch_with(&attend_lanes_kernel<TYPE, D, 2>, a, 2, joint_lds<2, D>(a, a.waves), two, s);
    if constexpr (TYPE == 0) return launch_columns<TYPE, D, 0>(a, s);
    if constexpr (TYPE == 1) return a.type == 1 ? launch_columns<TYPE, D, 1>(a, s) : launch_columns<TYPE, D, 0>(a, s);
    if constexpr (TYPE == 2 || TYPE == 3) return a.type == 2 ? launch_columns<TYPE, D, 1>(a, s) : launch_columns<TYPE, D, 3>(a, s);
    return hipErrorInvalidValue;  // launch_attend_parts has them
}

template <int TYPE>
hipError_t launch_split_width(const SplitArgs &a, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    if (w <= 64) return launch_split<TYPE, 64>(a, s);
    if (w <= 128) return launch_split<TYPE, 128>(a, s);
    return launch_split<TYPE, 256>(a, s);
}

}  // namespace

bool split_widths_ok(int qk, int vd) { return qk > 0 && vd > 0 && qk % 16 == 0 && vd % 16 == 0 && qk <= 256 && vd <= 256; }

int split_tile_columns(const SplitArgs &a, int cus) {
    const long long cols = static_cast<long long>(a.t) * a.group;
    if (a.pos && a.t > 1) return cols > kCols && std::max(a.c.qk, a.c.vd) <= 128 ? 2 * kCols : kCols;  // columns that see different keys
    if (cols <= 2) return static_cast<int>(cols);
    // Two columns a workgroup on the vector units for little work, 512 keys a CU
    // over the pairs of columns, of narrow heads of 16-bit and int8 caches: the
    // keys are read again from the L2, but a list's products leave one CU's
    // matrix units (one stream of 200 int8 keys, 8 heads of 48 over 2: 6.9 us
    // against 7.8; 32 of 448: 8.6 against 9.8; of 4000: 26.7 against 20.7;
    // float32 9.7 against 9.5, heads of 128 up to half as long again).
    const bool narrow = std::max(a.c.qk, a.c.vd) <= 64 && a.c.type != 0;
    const long long pairs = (cols + 1) / 2 * a.batch * a.c.kv_heads;
    // The weights of a list are summed over its heads by the workgroup that has them all.
    return narrow && !a.acc_out && pairs * a.nk_max <= 512LL * cus ? 2 : kCols;
}

int split_max_waves(const SplitArgs &a) {
    const int w = std::max(a.c.qk, a.c.vd);
    return w <= 128 ? 8 : 4;
}

bool split_weights_in_lds(const SplitArgs &a, int waves) {
    const int w = std::max(a.c.qk, a.c.vd), group = a.heads / a.c.kv_heads;
    const auto joint = [&](auto d) {
        constexpr int kD = decltype(d)::value;
        return a.tile == 1 ? Joint<1, kD>::floats(waves) : a.tile == 2 ? Joint<2, kD>::floats(waves) : Joint<kCols, kD>::floats(waves);
    };
    const int floats = w <= 64    ? joint(std::integral_constant<int, 64>{})
                       : w <= 128 ? joint(std::integral_constant<int, 128>{})
                                  : joint(std::integral_constant<int, 256>{});
    return a.t == 1 && group <= a.tile && sizeof(float) * (floats + group * static_cast<size_t>(a.nk_max)) <= kMostLds / 2;
}

hipError_t launch_attend_join(const SplitArgs &a, hipStream_t s) {
    const int blocks = (a.c.vd + 127) / 128;
    const long long grid = static_cast<long long>(a.batch) * a.t * a.heads * blocks;
    hipLaunchKernelGGL(attend_join_kernel, dim3(static_cast<unsigned>(grid)), dim3(64), 0, s, a, blocks);
    return hipGetLastError();
}

hipError_t launch_attend_split(const SplitArgs &a, hipStream_t s) {
    hipError_t e;
    if (a.tile > 2 && ((a.pos && a.t > 1) || a.c.type >= 4)) {
        e = launch_attend_parts(a, s);
    } else {
        switch (a.c.type) {
            case 0: e = launch_split_width<0>(a, s); break;
            case 1: e = launch_split_width<1>(a, s); break;
            case 2: e = launch_split_width<2>(a, s); break;
            case 3: e = launch_split_width<3>(a, s); break;
            case 4: e = launch_split_width<4>(a, s); break;
            default: e = launch_split_width<5>(a, s); break;
        }
    }
    if (e != hipSuccess || !a.part) return e;
    if ((e = launch_attend_join(a, s)) != hipSuccess) return e;
    if (a.acc_out && a.logits) {
        const int blocks = (a.nk_max + 255) / 256;
        hipLaunchKernelGGL(attend_weights_kernel, dim3(static_cast<unsigned>(a.batch) * a.c.kv_heads * blocks),
                           dim3(256), sizeof(float) * 2 * (a.heads / a.c.kv_heads), s, a, blocks);
    }
    return hipGetLastError();
}

}  // namespace cqhip
