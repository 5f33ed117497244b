// gfx950 attention of few query columns over paged caches, split over the
// keys' length: causal rows (kv_attend_rows_paged_dev of few rows), and one token
// a stream over caches with a scale a page (kv_attend_paged_dev).
//
// The split, the parts and the lanes' places are attend_split_kernel's; here the
// second product is one of 16 bits too. S = K q^T leaves key 4c + i of a step in
// register i of lane (column, c), and the lane's eight keys of two steps are the
// operand of v_mfma_f32_16x16x32 against the same keys' values: pairs of rows
// of the lane's piece (one exchange a pair), codes widened to bfloat16, exactly. The
// weights, times their key's scale, go in as three parts of 16 bits whose sum they
// are, so the sums are float32's. v_mfma_f32_16x16x4_f32 took 1024 cycles for 16
// keys of 128 values, these 192 (4 streams of 65,000 e4m3 keys 175 -> 106 us a call).
// Two tiles of 16 columns share the keys' and values' registers where there are more than 16.
#include "split_device.hpp"

#include <algorithm>
#include <type_traits>

namespace cqhip {
namespace {

// A float32 weight in three parts of 16 bits whose sum it is: of bfloat16 (the
// upper halves, and of what they leave), or of float16, of a weight that is lifted
// by 2^14 (towards 0, and of what they leave; none loses more than 2^-38 of 1).
constexpr float kPartLift = 16384.0f;
template <int TYPE>
__device__ __forceinline__ void weight_parts(float x, float y, uint32_t (&w)[3]) {
    if constexpr (TYPE == 1) {
        using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
        x *= kPartLift;
        y *= kPartLift;
#pragma unroll
        for (int z = 0; z < 3; ++z) {
            w[z] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
            const f16x2 h = __builtin_bit_cast(f16x2, w[z]);
            x -= static_cast<float>(h[0]);
            y -= static_cast<float>(h[1]);
        }
    } else {
#pragma unroll
        for (int z = 0; z < 3; ++z) {
            w[z] = upper_pair(x, y);
            x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
            y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
        }
    }
}

// Two e4m3 codes of a word (its upper two if hi) as bfloat16, exactly.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}

// Elements e (even) and e + 1 of a piece as a pair of the products' 16-bit type.
template <int TYPE>
__device__ __forceinline__ uint32_t pair_of(const uint32_t *w, int e) {
    if constexpr (TYPE == 4) return e4m3_pair(w[e / 4], e & 2);
    if constexpr (kScaled<TYPE>) return upper_pair(piece_value<TYPE>(w, e), piece_value<TYPE>(w, e + 1));
    return w[e / 2];
}

// Element e (even) and e + 1 of two value rows as pairs of the products' 16-bit
// type: (x[e], y[e]) and (x[e + 1], y[e + 1]); codes widened to bfloat16, exactly.
template <int TYPE>
__device__ __forceinline__ void row_pairs(const uint32_t *x, const uint32_t *y, int e, uint32_t &even, uint32_t &odd) {
    if constexpr (TYPE == 5) {
        even = upper_pair(piece_value<TYPE>(x, e), piece_value<TYPE>(y, e));
        odd = upper_pair(piece_value<TYPE>(x, e + 1), piece_value<TYPE>(y, e + 1));
    } else {
        even = __builtin_amdgcn_perm(pair_of<TYPE>(y, e), pair_of<TYPE>(x, e), 0x05040100);
        odd = __builtin_amdgcn_perm(pair_of<TYPE>(y, e), pair_of<TYPE>(x, e), 0x07060302);
    }
}

// TYPE: the cache's type; D: widths up to D (64, 128, 256); PARTS: 16-bit
// parts of a query value (0: the products of the logits in float32); TILES: of
// 16 columns; CAUSAL: columns at different positions, which see different keys.
template <int TYPE, int D, int PARTS, int TILES, bool CAUSAL>
__global__ __launch_bounds__(D <= 128 ? 512 : 256) void attend_parts_kernel(SplitArgs a, int col_tiles) {
    constexpr int kSize = kValueSize<TYPE>;
    constexpr int kPer = 16 / kSize;          // elements of a 16-byte piece of a key row
    constexpr int kPieces = D / (4 * kPer);   // pieces of a key row a lane loads
    constexpr int kVals = D / 16;             // elements of a lane's piece of a value row
    constexpr int kVWords = kVals * kSize / 4;
    constexpr int kSub = D * kSize <= 256 ? 2 : 1;  // 16-key steps of a tile
    constexpr int kTile = 16 * kSub;
    constexpr int kColumns = kCols * TILES;
    constexpr bool kParts16 = TYPE != 0;      // the second product in 16 bits
    // A tile's values are asked for a tile ahead too, where the registers of two
    // wavefronts a SIMD hold them (codes, two tiles of columns).
    constexpr bool kAhead = kScaled<TYPE> && TILES == 2;
    // How far logits may pass the maximum before sums and outputs are scaled to
    // a new one: by 2^8, but not in float16, whose lift leaves no room.
    constexpr float kLag = TYPE == 1 ? 0.0f : 8.0f;
    extern __shared__ __align__(16) float smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, c = lane >> 4;
    const Place p = place_of(a, col_tiles, kColumns);
    if (!p.ok) return;
    const Joint<kColumns, D> jt(smem, waves);
    // this lane's columns: query row col / group, head col % group of the group
    int col[TILES], col_pos[TILES];
    bool col_ok[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        col[t] = p.ct * kColumns + 16 * t + r;
        col_ok[t] = col[t] < p.cols;
        col_pos[t] = CAUSAL ? a.pos[p.b] + (col_ok[t] ? col[t] : p.cols - 1) / p.group : 0;
    }

    // Row of the lane's key of a tile (its first kTile lanes; keys past the part's last read that one's row).
    // Rows are looked up two tiles ahead, keys loaded one ahead, scales too; the
    // first ones' page table entries are asked for before the queries.
    auto row_of = [&](int j) { return array_row(a, p, min(j + (lane & (kTile - 1)), p.j1 - 1)); };
    const int step = waves * kTile;
    int j = p.j0 + wave * kTile, rows = 0, rows_next = 0;
    if (j < p.j1) {
        rows = row_of(j);
        rows_next = row_of(j + step);
    }

    // The query's pieces: in float32 with 1/scale and log2(e) folded in, or in
    // 16-bit parts of eight. All of them are asked for before any is looked at.
    constexpr int kEights = PARTS ? kPer / 8 : 1;
    float qv[TILES][PARTS ? 1 : kPieces * kPer];
    uint32_t qp[TILES][PARTS ? PARTS : 1][kPieces][kEights][4];
    {
        float x[TILES][kPieces][kPer];
        auto load_all = [&](auto vec) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const long long qo = query_at(a, p, col_ok[t] ? col[t] : 0);
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int d0 = (4 * k + c) * kPer;
                    load_query_values<kPer, decltype(vec)::value>(x[t][k], a, qo + (d0 < a.c.qk ? d0 : 0));
                }
            }
        };
        if (a.q_vec)
            load_all(std::true_type{});
        else
            load_all(std::false_type{});
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const bool ok = col_ok[t] && (4 * k + c) * kPer < a.c.qk;
                float (&y)[kPer] = x[t][k];
#pragma unroll
                for (int e = 0; e < kPer; ++e) y[e] = ok ? y[e] : 0.0f;
                if constexpr (PARTS == 0) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) qv[t][k * kPer + e] = y[e] * a.scale_log2;
                } else if constexpr (TYPE == 1) {  // a float16 query
#pragma unroll
                    for (int e = 0; e < kPer; e += 2)
                        qp[t][0][k][e / 8][e / 2 % 4] =
                            __builtin_bit_cast(uint16_t, static_cast<_Float16>(y[e])) |
                            static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(y[e + 1]))) << 16;
                } else {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) y[e] = __builtin_canonicalizef(y[e]);  // a NaN's mark in the upper half
#pragma unroll
                    for (int z = 0; z < PARTS; ++z)
#pragma unroll
                        for (int e = 0; e < kPer; e += 2) {
                            qp[t][z][k][e / 8][e / 2 % 4] = upper_pair(y[e], y[e + 1]);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {  // what the part leaves: nothing of an infinity
                                const float part = __uint_as_float(__float_as_uint(y[e + i]) & 0xffff0000u);
                                y[e + i] = fabsf(part) < INFINITY ? y[e + i] - part : 0.0f;
                            }
                        }
                }
            }
    }

    f32x4 o[TILES][kVals];
    float m[TILES], l[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int e = 0; e < kVals; ++e) o[t][e] = f32x4{0, 0, 0, 0};
        m[t] = -INFINITY;
        l[t] = 0.0f;
    }

    const unsigned char *kp = a.c.k + static_cast<long long>(p.h) * a.k_head, *vp = a.c.v + static_cast<long long>(p.h) * a.v_head;
    const int v_piece = r * kVals < a.c.vd ? r * (kVals * kSize) : 0;  // past the width: outputs that nothing reads

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
    auto load_values = [&](uint32_t (&x)[kSub][4][kVWords], int rows) {
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long row = __shfl(rows, 16 * s + 4 * c + i);
                load_words<kVWords>(x[s][i], vp + row * a.v_row + v_piece);
            }
    };
    // The scales of the lane's key of a tile.
    auto load_scales = [&](float (&x)[2], int rows) {
        if constexpr (kScaled<TYPE>) {
            x[0] = a.c.ks[scale_at(a, rows, p.h)];
            x[1] = a.c.vs[scale_at(a, rows, p.h)];
        }
    };

    float *lg = CAUSAL ? nullptr : a.logits;
    if (lg) lg += ((static_cast<long long>(p.b) * a.c.kv_heads + p.h) * p.group + (col_ok[0] ? col[0] : 0)) * a.nk_max;
    if (j < p.j1) {
        uint32_t kw[kSub][kPieces][4];
        float scales[2] = {1.0f, 1.0f};
        load_keys(kw, rows);
        load_scales(scales, rows);
        uint32_t va[kAhead ? kSub : 1][4][kVWords];
        if constexpr (kAhead) load_values(va, rows);
        for (; j < p.j1; j += step) {
            const int jn = j + step;
            uint32_t vw[kSub][4][kVWords];
            if constexpr (kAhead) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int k = 0; k < kVWords; ++k) vw[s][i][k] = va[s][i][k];
                if (jn < p.j1) load_values(va, rows_next);
            } else {
                load_values(vw, rows);
            }
            int rows_after = rows_next;
            if (jn + step < p.j1) rows_after = row_of(jn + step);

            f32x4 sc[TILES][kSub];
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int s = 0; s < kSub; ++s) sc[t][s] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
                if constexpr (PARTS == 0) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
#pragma unroll
                        for (int s = 0; s < kSub; ++s)
#pragma unroll
                            for (int t = 0; t < TILES; ++t)
                                sc[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(kw[s][k], e), qv[t][k * kPer + e],
                                                                                sc[t][s], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < kEights; ++e)
#pragma unroll
                        for (int s = 0; s < kSub; ++s) {
                            uint32_t ka[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) ka[z] = pair_of<TYPE>(kw[s][k], 8 * e + 2 * z);
#pragma unroll
                            for (int z = 0; z < PARTS; ++z)
#pragma unroll
                                for (int t = 0; t < TILES; ++t) sc[t][s] = mfma_16x16x32<TYPE>(ka, qp[t][z][k][e], sc[t][s]);
                        }
                }
            // An infinite key times a part of 0 is NaN: such logits again, in float32.
            if constexpr (PARTS == 3 && !kScaled<TYPE>) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    bool nan = false;
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i) nan |= sc[t][s][i] != sc[t][s][i];
                    if (__any(nan)) {
                        f32x4 y[kSub];
#pragma unroll
                        for (int s = 0; s < kSub; ++s) y[s] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int k = 0; k < kPieces; ++k)
#pragma unroll
                            for (int e = 0; e < kPer; ++e) {
                                const float q = (piece_value<2>(qp[t][0][k][e / 8], e & 7) + piece_value<2>(qp[t][1][k][e / 8], e & 7)) +
                                                piece_value<2>(qp[t][2][k][e / 8], e & 7);
#pragma unroll
                                for (int s = 0; s < kSub; ++s)
                                    y[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(kw[s][k], e), q, y[s], 0, 0, 0);
                            }
#pragma unroll
                        for (int s = 0; s < kSub; ++s)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sc[t][s][i] = sc[t][s][i] != sc[t][s][i] ? y[s][i] : sc[t][s][i];
                    }
                }
            }
            float ksc[kSub][4], vsc[kSub][4];
            if constexpr (kScaled<TYPE>) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ksc[s][i] = __shfl(scales[0], 16 * s + 4 * c + i) * (PARTS ? a.scale_log2 : 1.0f);
                        vsc[s][i] = __shfl(scales[1], 16 * s + 4 * c + i);
                    }
            }
            if (jn < p.j1) {
                load_keys(kw, rows_next);
                load_scales(scales, rows_next);
            }
            // past the last key values of 0, not that key's: a weight of 0 times an infinity
            if (!kFinite<TYPE> && j + kTile > p.j1) {
                asm volatile("" ::: "memory");  // a branch: as selects it is paid by every tile
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (j + 16 * s + 4 * c + i >= p.j1) {
#pragma unroll
                            for (int k = 0; k < kVWords; ++k) vw[s][i][k] = 0;
                        }
            }
            // whether all of the tile's columns see all of its keys
            bool all = j + kTile <= p.j1;
            if constexpr (CAUSAL) {
                const int lo = p.kl.row(j), hi = p.kl.row(min(j + kTile, p.j1) - 1);
                all = all && hi <= p.pos0 && (a.window == 0 || lo > p.pos1 - a.window || hi < a.sink);
            }
            uint32_t parts[TILES][kParts16 ? 3 : 1][4] = {};
            float w[TILES][kSub][4];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                float mt = -INFINITY;
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = sc[t][s][i];
                        if constexpr (kScaled<TYPE>)
                            x *= ksc[s][i];
                        else if constexpr (PARTS > 0)
                            x *= a.scale_log2;
                        sc[t][s][i] = x;
                    }
                if (!all) {
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int jj = j + 16 * s + 4 * c + i;
                            const bool seen = (jj < p.j1) & (!CAUSAL || sees_row(a, col_pos[t], p.kl.row(jj)));
                            sc[t][s][i] = seen ? sc[t][s][i] : -INFINITY;
                        }
                }
                if (!CAUSAL && a.acc_out && col_ok[t]) {
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int jj = j + 16 * s + 4 * c + i;
                            if (jj >= p.j1) continue;
                            if (lg)
                                lg[p.kl.row(jj)] = sc[t][s][i];
                            else
                                jt.logits[r * a.nk_max + jj] = sc[t][s][i];
                        }
                }
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mt = fmaxf(mt, sc[t][s][i]);
                mt = fmaxf(mt, xor_lane<16>(mt));
                mt = fmaxf(mt, xor_lane<32>(mt));
                if (__any(mt > m[t] + kLag)) {
                    const float mn = fmaxf(m[t], mt);
                    const float f = m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[t] - mn);
                    m[t] = mn;
                    l[t] *= f;
#pragma unroll
                    for (int e = 0; e < kVals; ++e) o[t][e] *= f;
                }
                const float mu = m[t] == -INFINITY ? 0.0f : m[t];  // no key above -inf so far: every weight 0
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[t][s][i] = __builtin_amdgcn_exp2f(sc[t][s][i] - mu);
                        l[t] += w[t][s][i];
                        if constexpr (kScaled<TYPE>) w[t][s][i] = all || j + 16 * s + 4 * c + i < p.j1 ? w[t][s][i] * vsc[s][i] : 0.0f;
                    }
                if constexpr (kParts16) {
                    // a contraction of 32: the lane's keys 4 c + i of both steps of 16
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            uint32_t z[3];
                            weight_parts<TYPE>(w[t][s][i], w[t][s][i + 1], z);
#pragma unroll
                            for (int k = 0; k < 3; ++k) parts[t][k][2 * s + i / 2] = z[k];
                        }
                }
            }
            if constexpr (kParts16) {
#pragma unroll
                for (int e = 0; e < kVals; e += 2) {
                    uint32_t even[4] = {}, odd[4] = {};
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) row_pairs<TYPE>(vw[s][i], vw[s][i + 1], e, even[2 * s + i / 2], odd[2 * s + i / 2]);
#pragma unroll
                    for (int k = 0; k < 3; ++k)
#pragma unroll
                        for (int t = 0; t < TILES; ++t) {
                            o[t][e] = mfma_16x16x32<TYPE>(even, parts[t][k], o[t][e]);
                            o[t][e + 1] = mfma_16x16x32<TYPE>(odd, parts[t][k], o[t][e + 1]);
                        }
                }
            } else {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < kVals; ++e)
#pragma unroll
                            for (int t = 0; t < TILES; ++t)
                                o[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece_value<TYPE>(vw[s][i], e), w[t][s][i], o[t][e], 0, 0, 0);
            }
            rows = rows_next;
            rows_next = rows_after;
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        l[t] += xor_lane<16>(l[t]);
        l[t] += xor_lane<32>(l[t]);
        if (c == 0) {
            jt.ml[(wave * 2) * kColumns + 16 * t + r] = m[t];
            jt.ml[(wave * 2 + 1) * kColumns + 16 * t + r] = l[t];
        }
        if (col_ok[t]) {
#pragma unroll
            for (int e = 0; e < kVals; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    jt.o[(wave * kColumns + 16 * t + r) * jt.kRow + kVals * (4 * c + i) + e] =
                        TYPE == 1 ? o[t][e][i] * (1.0f / kPartLift) : o[t][e][i];
        }
    }
    finish<kColumns, D, TYPE>(a, p, jt);
}

template <int TYPE, int D, int PARTS, int TILES, bool CAUSAL>
hipError_t launch_tiles(const SplitArgs &a, hipStream_t s) {
    static std::atomic<unsigned long long> attr{0};
    return launch_with(&attend_parts_kernel<TYPE, D, PARTS, TILES, CAUSAL>, a, kCols * TILES, joint_lds<kCols * TILES, D>(a, a.waves),
                       attr, s);
}

template <int TYPE, int D, int PARTS>
hipError_t launch_parts(const SplitArgs &a, hipStream_t s) {
    if (a.pos) {
        if constexpr (D <= 128)
            if (a.tile == 2 * kCols) return launch_tiles<TYPE, D, PARTS, 2, true>(a, s);
        return launch_tiles<TYPE, D, PARTS, 1, true>(a, s);
    }
    if constexpr (TYPE >= 4) return launch_tiles<TYPE, D, PARTS, 1, false>(a, s);
    return hipErrorInvalidValue;
}

template <int TYPE, int D>
hipError_t launch_query(const SplitArgs &a, hipStream_t s) {
    if constexpr (TYPE == 0) return launch_parts<TYPE, D, 0>(a, s);
    if constexpr (TYPE == 1) return a.type == 1 ? launch_parts<TYPE, D, 1>(a, s) : launch_parts<TYPE, D, 0>(a, s);
    if constexpr (TYPE >= 2) return a.type == 2 ? launch_parts<TYPE, D, 1>(a, s) : launch_parts<TYPE, D, 3>(a, s);
}

template <int TYPE>
hipError_t launch_width(const SplitArgs &a, hipStream_t s) {
    const int w = std::max(a.c.qk, a.c.vd);
    return w <= 64 ? launch_query<TYPE, 64>(a, s) : w <= 128 ? launch_query<TYPE, 128>(a, s) : launch_query<TYPE, 256>(a, s);
}

}  // namespace

hipError_t launch_attend_parts(const SplitArgs &a, hipStream_t s) {
    switch (a.c.type) {
        case 0: return launch_width<0>(a, s);
        case 1: return launch_width<1>(a, s);
        case 2: return launch_width<2>(a, s);
        case 4: return launch_width<4>(a, s);
        default: return launch_width<5>(a, s);
    }
}

}  // namespace cqhip
