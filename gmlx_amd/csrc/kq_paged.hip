// Attention of each row's new tokens over a paged KV cache (kq_sdpa_paged).
//
// A row's new tokens and the G = Hq / Hkv query heads that share a kv head are
// flattened to n * G query columns (column c: token c / G, head c % G).  Both
// products run on v_mfma_f32_16x16x32 with the query columns in the MFMA's
// columns:
//   S^T[tok, col] = K[tok, d] . q^T[d, col],  O^T[d, col] += V^T[d, tok] . P^T[tok, col]
// so that a lane's scores are the P.V operand it needs (lane 16 g + r holds
// column r at tokens 4g .. 4g+3 of each 16), and the softmax statistics of a
// column live in the four lanes that hold it.
#include "kq_paged.h"

namespace {

struct PagedArgs {
    const uint16_t *q;
    uint16_t *out;
    const void *k, *v;
    const uint16_t *ks, *kb, *vs, *vb;
    const int32_t *table, *kv_lens, *cu_q;
    int64_t q_stride, out_stride, page_stride, head_stride, table_stride;
    int32_t tok_stride, lps, n_pages, width;
    int32_t T, B, Hq, Hkv, G, max_q, max_kv;
    float scale_log2;
    float *part, *ml;  // split partials: [slot][D] sums, [slot][2] (maximum, sum)
};

constexpr int kSplitTokens = 512;   // least keys of a split
constexpr int kSplitWaves = 2048;   // waves of a row that splitting aims at

// Splits of a row of n tokens and kv keys: from the row and the head counts
// alone, so that a row of a batch has the bits of the row alone.
__host__ __device__ __forceinline__ int paged_splits(int n, int kv, int G, int Hkv) {
    const int waves = (int)(((int64_t)n * G + 15) / 16) * Hkv;
    if (waves == 0) return 1;
    const int most = (kv + kSplitTokens - 1) / kSplitTokens;
    const int want = (kSplitWaves + waves - 1) / waves;
    return max(1, min(want, most));
}

struct Row {
    int q0;       // first query row
    int n, full;  // tokens computed, tokens of the row
    int kv;       // keys
    int blocks, splits;
};

__device__ __forceinline__ Row row_at(const PagedArgs &a, int b) {
    Row r;
    r.q0 = min(max(a.cu_q[b], 0), a.T);
    r.full = min(max(a.cu_q[b + 1], r.q0), a.T) - r.q0;
    r.n = min(r.full, a.max_q);
    r.kv = (int)min((int64_t)max(min(a.kv_lens[b], a.max_kv), 0), (int64_t)a.width << a.lps);
    r.blocks = (int)(((int64_t)r.n * a.G + 15) / 16);
    r.splits = paged_splits(r.n, r.kv, a.G, a.Hkv);
    return r;
}

__device__ __forceinline__ int64_t row_units(const PagedArgs &a, const Row &r) {
    return (int64_t)r.blocks * r.splits * a.Hkv;
}

__device__ __forceinline__ int64_t row_slots(const PagedArgs &a, const Row &r) {
    return r.splits > 1 ? (int64_t)r.n * a.Hq * r.splits : 0;
}

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lane = kq_lane();
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t t = __shfl_up(v, off);
        if (lane >= off) v += t;
    }
    return v;
}

// The row that unit u belongs to, with u made its number within the row and
// the row's first partial slot; false past the last unit.  The unit counts are
// summed over the rows, 64 at a time, by every wave that asks.
__device__ __forceinline__ bool find_unit(const PagedArgs &a, int64_t &u, int &b, Row &r, int64_t &slot0) {
    const int lane = kq_lane();
    int64_t slots = 0;
    for (int c0 = 0; c0 < a.B; c0 += 64) {
        const int row = c0 + lane;
        int64_t mu = 0, ms = 0;
        if (row < a.B) {
            const Row x = row_at(a, row);
            mu = row_units(a, x);
            ms = row_slots(a, x);
        }
        const int64_t iu = wave_scan(mu), is = wave_scan(ms);
        const int64_t total = __shfl(iu, 63);
        if (u < total) {
            const int src = __builtin_ctzll(__ballot(u < iu));
            b = __builtin_amdgcn_readfirstlane(c0 + src);
            u -= __shfl(iu - mu, src);
            slot0 = slots + __shfl(is - ms, src);
            r = row_at(a, b);
            return true;
        }
        u -= total;
        slots += __shfl(is, 63);
    }
    return false;
}

// Exponent shift of the probabilities: they and their sum are 2^kShift times
// the softmax's, which keeps fp16 ones of far smaller keys out of the
// subnormals; the quotient is the same.  An 8-bit cache multiplies a
// probability by its key's scale (up to 514) before it is rounded.
template <bool BF, bool Q8>
constexpr float shift() { return BF ? 0.f : Q8 ? 6.f : 10.f; }

template <int D>
struct Geo {
    static constexpr int TT = D > 256 ? 16 : 32;  // tokens a tile
    static constexpr int CH = TT / 16;            // 16-token chunks
    static constexpr int VT = TT / 4;             // V rows a lane
    static constexpr int NC = D / 32;             // 32-wide pieces of the head dim
};

// Where a tile's chunks start in the pool (elements or bytes; uniform), and
// which of them lie in a page of the pool.
template <int D>
struct TileAt {
    int64_t off[Geo<D>::CH];
    bool ok[Geo<D>::CH];
};

// One tile in registers, 16-bit pool.
template <int D, bool BF>
struct Tile16 {
    static constexpr int CH = Geo<D>::CH, VT = Geo<D>::VT, NC = Geo<D>::NC, NG = (D + 127) / 128;
    u32x4 k[CH][NC];  // token 16 ch + r, d = 32 c + 8 g .. +7
    u32x4 v[NG][VT];  // token 4g + i | 16 + 4g + i - 4, d = 128 dg + 8 r .. +7

    __device__ __forceinline__ void load(const PagedArgs &a, const TileAt<D> &at) {
        const int lane = kq_lane(), r = lane & 15, g = lane >> 4;
        const uint32_t ko = (uint32_t)(r * a.tok_stride + 8 * g);
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
            const uint16_t *kp = (const uint16_t *)a.k + at.off[ch];
#pragma unroll
            for (int c = 0; c < NC; ++c) k[ch][c] = *(const u32x4 *)(kp + (ko + 32 * c));
        }
#pragma unroll
        for (int dg = 0; dg < NG; ++dg) {
            const uint32_t d0 = min(128 * dg + 8 * r, D - 8);
#pragma unroll
            for (int i = 0; i < VT; ++i) {
                const uint16_t *vp = (const uint16_t *)a.v + at.off[i >> 2];
                v[dg][i] = *(const u32x4 *)(vp + ((uint32_t)((4 * g + (i & 3)) * a.tok_stride) + d0));
            }
        }
    }
};

// 8 bytes as 16-bit floats of their integer values less Z (0 or 128), exactly.
template <bool BF, int Z>
__device__ __forceinline__ u32x4 bytes8(u32x2 q) {
    if constexpr (!BF) {
        const half2_t z = {(_Float16)(1024.f + Z), (_Float16)(1024.f + Z)};
        auto pair = [&](uint32_t w, uint32_t sel) {
            return __builtin_bit_cast(uint32_t, kq_as_h2(kq_bytes_to_h2_biased(w, sel)) - z);
        };
        return u32x4{pair(q.x, KQ_SEL_B01), pair(q.x, KQ_SEL_B23), pair(q.y, KQ_SEL_B01), pair(q.y, KQ_SEL_B23)};
    } else {
        // fp32 values of at most 8 significant bits: their upper halves are
        // the bf16 values
        auto pair = [&](uint32_t w, int j) {
            const float x = (float)((w >> (8 * j)) & 0xFFu) - (float)Z, y = (float)((w >> (8 * j + 8)) & 0xFFu) - (float)Z;
            return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
        };
        return u32x4{pair(q.x, 0), pair(q.x, 2), pair(q.y, 0), pair(q.y, 2)};
    }
}

template <int SG>
struct GroupWords;  // SG 16-bit values at 2-byte alignment
template <>
struct GroupWords<1> { typedef uint16_t type; };
template <>
struct GroupWords<2> { typedef u32_a2 type; };
template <>
struct GroupWords<4> { typedef u32x2_a2 type; };
template <>
struct GroupWords<8> { typedef u32x4_a2 type; };

// One tile of an 8-bit pool.  The products run on the integers: with k = s q +
// b for a group of 64,
//   q . k = sum over groups of s (q . int_k) + b (sum of q),
//   P . V = sum of (P s) int_v + sum of P b,
// the scales of a lane's tokens being those of its scores, so nothing is
// dequantised and no dequantised value is rounded.  V's integers are centred
// (less 128, b + 128 s for b) to halve what the rounding of P s costs.
template <int D, bool BF>
struct Tile8 {
    static constexpr int CH = Geo<D>::CH, VT = Geo<D>::VT, NC = Geo<D>::NC, SG = D / 64;
    typedef typename GroupWords<SG>::type W;
    static constexpr int NW = (SG + 1) / 2;
    u32x2 k[CH][NC];       // token 16 ch + r, d = 64 (c / 2) + 16 g + 8 (c % 2) .. +7
    uint32_t v[SG][VT];    // token as above, d = 64 grp + 4 r .. +3
    uint32_t ks[CH][4][NW], kb[CH][4][NW], vs[CH][4][NW], vb[CH][4][NW];  // tokens 16 ch + 4g .. +3

    __device__ __forceinline__ static void words(const uint16_t *p, uint32_t (&w)[NW]) {
        if constexpr (SG == 1) w[0] = *p;
        else {
            const W x = *(const W *)p;
            __builtin_memcpy(w, &x, sizeof(w));
        }
    }
    // scale of group grp
    __device__ __forceinline__ static float of(const uint32_t (&w)[NW], int grp) {
        return f16bits_to_f32<BF>(grp & 1 ? w[grp >> 1] >> 16 : w[grp >> 1] & 0xFFFFu);
    }
    __device__ __forceinline__ void load(const PagedArgs &a, const TileAt<D> &at) {
        const int lane = kq_lane(), r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
            const uint8_t *kp = (const uint8_t *)a.k + at.off[ch];
#pragma unroll
            for (int i = 0; i < NC / 2; ++i) {
                const u32x4 w = *(const u32x4 *)(kp + (uint32_t)(r * D + 64 * i + 16 * g));
                k[ch][2 * i] = u32x2{w.x, w.y};
                k[ch][2 * i + 1] = u32x2{w.z, w.w};
            }
            const int64_t s0 = at.off[ch] >> 6;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t so = (uint32_t)((4 * g + i) * SG);
                words(a.ks + s0 + so, ks[ch][i]);
                words(a.kb + s0 + so, kb[ch][i]);
                words(a.vs + s0 + so, vs[ch][i]);
                words(a.vb + s0 + so, vb[ch][i]);
            }
        }
#pragma unroll
        for (int grp = 0; grp < SG; ++grp)
#pragma unroll
            for (int i = 0; i < VT; ++i)
                v[grp][i] = *(const uint32_t *)((const uint8_t *)a.v + at.off[i >> 2] +
                                                (uint32_t)((4 * g + (i & 3)) * D + 64 * grp + 4 * r));
    }
};

// Query fragments and sums of one unit (16 query columns).
template <int D, bool BF, bool Q8>
struct State {
    static constexpr int NC = Geo<D>::NC, CH = Geo<D>::CH;
    static constexpr int NO = Q8 ? D / 16 : (D + 127) / 128 * 8;
    static constexpr int SG = Q8 ? D / 64 : 1;
    half8_t qf[NC];
    float qsum[SG];  // Q8: sum of the column's query over each group
    floatx4 o[NO];
    float bias[SG];  // Q8: this lane's share of sum of p b
    float m_run, l_part;
    int seen;  // keys that the column sees: 0 .. seen - 1

    // value 4 consecutive results start at: d of (o[j .. ], e)
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < SG; ++j) bias[j] = 0.f;
        m_run = -INFINITY;
        l_part = 0.f;
    }

    // Scores of the tile in log2 units.
    template <class Tile>
    __device__ __forceinline__ void scores(const Tile &t, float scale_log2, float (&s)[8]) {
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
            if constexpr (!Q8) {
                floatx4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < NC; ++c) acc = mfma<BF>(__builtin_bit_cast(half8_t, t.k[ch][c]), qf[c], acc);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * ch + e] = acc[e] * scale_log2;
            } else {
                float sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int grp = 0; grp < SG; ++grp) {
                    floatx4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 2 * grp; c < 2 * grp + 2; ++c)
                        acc = mfma<BF>(__builtin_bit_cast(half8_t, bytes8<BF, 0>(t.k[ch][c])), qf[c], acc);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sum[e] = fmaf(t.of(t.ks[ch][e], grp), acc[e], fmaf(t.of(t.kb[ch][e], grp), qsum[grp], sum[e]));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * ch + e] = sum[e] * scale_log2;
            }
        }
    }

    // MASK: some of the tile's keys are hidden from some column (vis: bit j for
    // this lane's j-th score).
    template <bool MASK, class Tile>
    __device__ __forceinline__ void tile(const Tile &t, float scale_log2, uint32_t vis) {
        float s[8];
        scores(t, scale_log2, s);
        constexpr int N = 4 * CH;
        if constexpr (MASK) {
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] = (vis >> j) & 1 ? s[j] : -INFINITY;
        }
        float tmax = s[0];
#pragma unroll
        for (int j = 1; j < N; ++j) tmax = fmaxf(tmax, s[j]);
        const float m_new = fmaxf(m_run, max_over_groups(tmax));
        // no key yet (only where MASK): every power below is 0, not exp(-inf + inf)
        const float m_use = MASK && m_new == -INFINITY ? 0.f : m_new;
        // arguments are at most 0: the hardware's flush of results below 2^-126
        // is far below the rounding of a sum that holds the row's maximum
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        float p[8], psum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = j < N ? __builtin_amdgcn_exp2f(s[j] - (m_use - shift<BF, Q8>())) : 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) psum += p[j];
        l_part = l_part * alpha + psum;
        m_run = m_new;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
            for (int j = 0; j < NO; ++j) o[j] = o[j] * alpha;
#pragma unroll
            for (int j = 0; j < SG; ++j) bias[j] *= alpha;
        }
        if constexpr (!Q8) {
            pv16<MASK>(t, p, vis);
        } else {
#pragma unroll
            for (int grp = 0; grp < SG; ++grp) {
                float ps[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j >= N) {
                        ps[j] = 0.f;
                        continue;
                    }
                    const float sc = t.of(t.vs[j >> 2][j & 3], grp), bi = t.of(t.vb[j >> 2][j & 3], grp);
                    // (a hidden key's scale and bias may be anything)
                    const bool on = !MASK || ((vis >> j) & 1);
                    ps[j] = on ? p[j] * sc : 0.f;
                    bias[grp] += on ? fmaf(128.f, ps[j], p[j] * bi) : 0.f;
                }
                const half8_t pf = __builtin_bit_cast(half8_t, u32x4{pack2<BF>(ps[0], ps[1]), pack2<BF>(ps[2], ps[3]),
                                                                     pack2<BF>(ps[4], ps[5]), pack2<BF>(ps[6], ps[7])});
                // byte j of tokens 0 .. 7 as one operand
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = i < Tile::VT ? t.v[grp][i] : 0x80808080u;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // (b0 b1 of two tokens) -> two words of one byte each of four tokens
                    const uint32_t sel = half ? 0x07030602u : 0x05010400u;
                    const uint32_t t01 = __builtin_amdgcn_perm(w[1], w[0], sel), t23 = __builtin_amdgcn_perm(w[3], w[2], sel);
                    const uint32_t t45 = __builtin_amdgcn_perm(w[5], w[4], sel), t67 = __builtin_amdgcn_perm(w[7], w[6], sel);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t pick = e ? 0x07060302u : 0x05040100u;
                        const u32x2 b8 = {__builtin_amdgcn_perm(t23, t01, pick), __builtin_amdgcn_perm(t67, t45, pick)};
                        const int j = grp * 4 + 2 * half + e;
                        o[j] = mfma<BF>(__builtin_bit_cast(half8_t, bytes8<BF, 128>(b8)), pf, o[j]);
                    }
                }
            }
        }
        kq_mfma_drain();
    }

    template <bool MASK, class Tile>
    __device__ __forceinline__ void pv16(const Tile &t, const float (&p)[8], uint32_t vis) {
        const half8_t pf = __builtin_bit_cast(half8_t, u32x4{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3]),
                                                             pack2<BF>(p[4], p[5]), pack2<BF>(p[6], p[7])});
        constexpr uint32_t kInf = BF ? 0x7F80u : 0x7C00u, kOne = BF ? 0x3F80u : 0x3C00u;
        bool odd = false;
        half8_t seen_f = pf;
        if constexpr (MASK) {
            // A hidden key's value times its probability 0 is NaN where the
            // value is an infinity or NaN: look for those, and where there are
            // any, take them out of the product and add them to the columns
            // that see them (products of 0 / 1 matrices).
#pragma unroll
            for (int dg = 0; dg < Tile::NG; ++dg)
#pragma unroll
                for (int i = 0; i < Tile::VT; ++i)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t x = t.v[dg][i][w];
                        odd |= (x & kInf) == kInf || (x & (kInf << 16)) == (kInf << 16);
                    }
            odd = __builtin_amdgcn_ballot_w64(odd) != 0;
            u32x4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                f[j] = ((vis >> (2 * j)) & 1 ? kOne : 0u) | ((vis >> (2 * j + 1)) & 1 ? kOne << 16 : 0u);
            seen_f = __builtin_bit_cast(half8_t, f);
        }
#pragma unroll
        for (int dg = 0; dg < Tile::NG; ++dg) {
            u32x4 vr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) vr[i] = i < Tile::VT ? t.v[dg][i] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                u32x4 f;
                f.x = __builtin_amdgcn_perm(vr[1][j >> 1], vr[0][j >> 1], sel);
                f.y = __builtin_amdgcn_perm(vr[3][j >> 1], vr[2][j >> 1], sel);
                f.z = __builtin_amdgcn_perm(vr[5][j >> 1], vr[4][j >> 1], sel);
                f.w = __builtin_amdgcn_perm(vr[7][j >> 1], vr[6][j >> 1], sel);
                if (MASK && odd) {
                    u32x4 up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t x = (f[w] >> (16 * half)) & 0xFFFFu;
                            const bool bad = (x & kInf) == kInf, nan = (x & 0x7FFFu) > kInf;
                            if (bad) {
                                f[w] &= half ? 0x0000FFFFu : 0xFFFF0000u;
                                if (nan || !(x & 0x8000u)) up[w] |= kOne << (16 * half);
                                if (nan || (x & 0x8000u)) down[w] |= kOne << (16 * half);
                            }
                        }
                    const floatx4 z = {0, 0, 0, 0};
                    const floatx4 a = mfma<BF>(__builtin_bit_cast(half8_t, up), seen_f, z);
                    const floatx4 b = mfma<BF>(__builtin_bit_cast(half8_t, down), seen_f, z);
                    kq_mfma_drain();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (a[e] > 0.f) o[dg * 8 + j][e] += INFINITY;
                        if (b[e] > 0.f) o[dg * 8 + j][e] -= INFINITY;
                    }
                }
                o[dg * 8 + j] = mfma<BF>(__builtin_bit_cast(half8_t, f), pf, o[dg * 8 + j]);
            }
        }
    }
};

// One wave a workgroup; unit = (row, 16-column block, split, kv head), the kv
// heads fastest (with eight of them, one per XCD: the blocks of a head share
// their keys in that XCD's L2).
template <int D, bool BF, bool Q8>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void kq_paged_split_kernel(
    PagedArgs a) {
    using Tile = std::conditional_t<Q8, Tile8<D, BF>, Tile16<D, BF>>;
    constexpr int TT = Geo<D>::TT, CH = Geo<D>::CH, NC = Geo<D>::NC;
    constexpr int NBUF = D >= 256 ? 1 : 2;
    const int lane = kq_lane(), r = lane & 15, g = lane >> 4;
    for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
        int64_t u = unit, slot0;
        int b;
        Row row;
        if (!find_unit(a, u, b, row, slot0)) return;
        const uint32_t nth = (uint32_t)u, rest = nth / (uint32_t)a.Hkv;
        const int h = (int)(nth - rest * a.Hkv);
        const int blk = (int)(rest / (uint32_t)row.splits), s = (int)(rest - (uint32_t)blk * row.splits);

        // this lane's column
        const int64_t col = (int64_t)blk * 16 + r;
        const bool live = col < (int64_t)row.n * a.G;
        const int i = live ? (int)(col / a.G) : row.n - 1, head = live ? (int)(col - (int64_t)i * a.G) : 0;
        const int hq = h * a.G + head;
        State<D, BF, Q8> st;
        st.init();
        const int first_i = (int)((int64_t)blk * 16 / a.G);
        const int last_i = min((int)(((int64_t)blk * 16 + 15) / a.G), row.n - 1);
        // keys seen: column i's, the block's least and most
        const auto seen_by = [&](int tok) { return max(row.kv - row.full + tok + 1, 0); };
        st.seen = live ? seen_by(i) : 0x7fffffff;
        const int least = __builtin_amdgcn_readfirstlane(seen_by(first_i));
        const int most = __builtin_amdgcn_readfirstlane(min(seen_by(last_i), row.kv));
        // whole tiles, about the same for each split
        const int per = ((row.kv + row.splits - 1) / row.splits + TT - 1) / TT * TT;
        const int t_begin = __builtin_amdgcn_readfirstlane(s * per);
        const int t_end = __builtin_amdgcn_readfirstlane(min(most, t_begin + per));
        const uint16_t *qp = a.q + (int64_t)(row.q0 + i) * a.q_stride + (int64_t)hq * D;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = Q8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
            const u32x4 w = *(const u32x4 *)(qp + d);
            st.qf[c] = __builtin_bit_cast(half8_t, live ? w : u32x4{0u, 0u, 0u, 0u});
        }
        if constexpr (Q8) {
#pragma unroll
            for (int grp = 0; grp < D / 64; ++grp) {
                float sum = 0.f;
#pragma unroll
                for (int c = 2 * grp; c < 2 * grp + 2; ++c) {
                    const u32x4 w = __builtin_bit_cast(u32x4, st.qf[c]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum += f16bits_to_f32<BF>(w[x] & 0xFFFFu) + f16bits_to_f32<BF>(w[x] >> 16);
                }
                sum += __shfl_xor(sum, 16);
                st.qsum[grp] = sum + __shfl_xor(sum, 32);
            }
        }

        if (t_end > t_begin) {
            // the row's block table, 64 entries at a time in a register
            const int32_t *tab = a.table + (int64_t)b * a.table_stride;
            const int sh = a.lps - 4;  // log2 of a page's chunks
            const int c_last = (t_end - 1) >> 4, p_last = c_last >> sh;
            int p0 = (t_begin >> 4) >> sh;
            int ids = tab[min(p0 + lane, p_last)];
            const int64_t h_off = (int64_t)h * a.head_stride;
            auto at_tile = [&](int t0) {
                TileAt<D> x;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) {
                    // (chunks past the end repeat the last: their keys are hidden)
                    const int c = min((t0 >> 4) + ch, c_last), p = c >> sh;
                    if (p - p0 >= 64) {
                        p0 = p;
                        ids = tab[min(p0 + lane, p_last)];
                    }
                    const int id = __builtin_amdgcn_readlane(ids, p - p0);
                    x.ok[ch] = (uint32_t)id < (uint32_t)a.n_pages;
                    x.off[ch] = uniform64((int64_t)(x.ok[ch] ? id : 0) * a.page_stride + h_off +
                                          (int64_t)((c - (p << sh)) * 16) * a.tok_stride);
                }
                return x;
            };
            Tile ring[NBUF];
            TileAt<D> at[NBUF];
#pragma unroll
            for (int j = 0; j < NBUF - 1; ++j) {
                at[j] = at_tile(t_begin + TT * j);
                ring[j].load(a, at[j]);
            }
            for (int t0 = t_begin; t0 < t_end; t0 += TT * NBUF) {
#pragma unroll
                for (int j = 0; j < NBUF; ++j) {
                    const int nx = (j + NBUF - 1) % NBUF;
                    at[nx] = at_tile(t0 + TT * (j + NBUF - 1));
                    ring[nx].load(a, at[nx]);
                    __builtin_amdgcn_sched_barrier(0);
                    const int t = t0 + TT * j;
                    if (t < t_end) {
                        bool whole = t + TT <= min(least, t_end);
#pragma unroll
                        for (int ch = 0; ch < CH; ++ch) whole &= at[j].ok[ch];
                        if (whole) {
                            st.template tile<false>(ring[j], a.scale_log2, 0);
                        } else {
                            const int lim = min(st.seen, t_end);
                            uint32_t vis = 0;
#pragma unroll
                            for (int x = 0; x < 4 * CH; ++x)
                                if (at[j].ok[x >> 2] && t + 16 * (x >> 2) + 4 * g + (x & 3) < lim) vis |= 1u << x;
                            st.template tile<true>(ring[j], a.scale_log2, vis);
                        }
                    }
                }
            }
        }

        float l = st.l_part + __shfl_xor(st.l_part, 16);
        l += __shfl_xor(l, 32);
        if constexpr (Q8) {
#pragma unroll
            for (int grp = 0; grp < D / 64; ++grp) {
                float x = st.bias[grp] + __shfl_xor(st.bias[grp], 16);
                x += __shfl_xor(x, 32);
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[grp * 4 + e] = st.o[grp * 4 + e] + x;
            }
        }
        if (!live) continue;
        const bool whole = row.splits == 1;
        const float mul = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
        uint16_t *op = a.out + (int64_t)(row.q0 + i) * a.out_stride + (int64_t)hq * D;
        const int64_t slot = slot0 + ((int64_t)i * a.Hq + hq) * row.splits + s;
        float *pp = a.part + slot * D;
        // runs of W consecutive values: lane (column, g), o[j0 .. j0 + W)[e]
        constexpr int W = Q8 ? 4 : 8;
#pragma unroll
        for (int j0 = 0; j0 < State<D, BF, Q8>::NO; j0 += W)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 16 * j0 + W * (4 * g + e);
                if (d >= D) continue;
                if (whole) {
                    uint32_t w[W / 2];
#pragma unroll
                    for (int x = 0; x < W / 2; ++x)
                        w[x] = (uint32_t)from_f32<BF>(st.o[j0 + 2 * x][e] * mul) |
                               ((uint32_t)from_f32<BF>(st.o[j0 + 2 * x + 1][e] * mul) << 16);
                    if constexpr (W == 8) *(u32x4 *)(op + d) = u32x4{w[0], w[1], w[2], w[3]};
                    else *(u32x2 *)(op + d) = u32x2{w[0], w[1]};
                } else {
#pragma unroll
                    for (int x = 0; x < W; x += 4)
                        *(float4 *)(pp + d + x) =
                            make_float4(st.o[j0 + x][e], st.o[j0 + x + 1][e], st.o[j0 + x + 2][e], st.o[j0 + x + 3][e]);
                }
            }
        if (!whole && g == 0) {
            a.ml[2 * slot] = st.m_run;
            a.ml[2 * slot + 1] = l;
        }
    }
}

// One wave a (token, query head) of a row with splits: rescales the splits to
// their common maximum and sums them in split order.
template <int D, bool BF>
__global__ __launch_bounds__(256) void kq_paged_merge_kernel(PagedArgs a) {
    constexpr int V = D >= 256 ? D / 64 : 2;  // values a lane
    const int lane = kq_lane();
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(item / a.Hq), hq = (int)(item - (int64_t)t * a.Hq);
    if (t >= a.T) return;
    // the token's row
    int64_t slot = 0;
    int splits = 0;
    for (int c0 = 0; c0 < a.B && !splits; c0 += 64) {
        const int row = c0 + lane;
        int64_t ms = 0;
        Row x{};
        if (row < a.B) {
            x = row_at(a, row);
            ms = row_slots(a, x);
        }
        const int64_t is = wave_scan(ms);
        const uint64_t hit = __ballot(row < a.B && t >= x.q0 && t < x.q0 + x.n);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            splits = __shfl(x.splits, src);
            slot += __shfl(is - ms, src) + ((int64_t)(t - __shfl(x.q0, src)) * a.Hq + hq) * splits;
        } else {
            slot += __shfl(is, 63);
        }
    }
    if (splits < 2) return;
    const float *ml = a.ml + 2 * slot;
    float m = -INFINITY;
    for (int s = lane; s < splits; s += 64) m = fmaxf(m, ml[2 * s]);
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    float acc[V], l = 0.f;
#pragma unroll
    for (int x = 0; x < V; ++x) acc[x] = 0.f;
    const int d = lane * V;
    if (d >= D) return;
    for (int s = 0; s < splits; ++s) {
        const float ms = ml[2 * s];
        const float ls = ml[2 * s + 1];
        const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
        if (f == 0.f && ls == ls) continue;  // (a split without keys holds zeros; one of NaN scores a NaN sum)
        l += f * ls;
        const float *p = a.part + (slot + s) * D + d;
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] += f * p[x];
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    uint16_t *op = a.out + (int64_t)t * a.out_stride + (int64_t)hq * D + d;
#pragma unroll
    for (int x = 0; x < V; ++x) op[x] = from_f32<BF>(acc[x] * inv);
}

template <int D, bool BF, bool Q8>
void launch_split(const PagedArgs &a, int grid, hipStream_t s) {
    hipLaunchKernelGGL((kq_paged_split_kernel<D, BF, Q8>), dim3(grid), dim3(64), 0, s, a);
}

template <int D, bool BF>
void launch(const PagedArgs &a, bool q8, int grid, bool merge, hipStream_t s) {
    if (q8) {
        if constexpr (D % 64 == 0) launch_split<D, BF, true>(a, grid, s);
    } else {
        launch_split<D, BF, false>(a, grid, s);
    }
    if (merge)
        hipLaunchKernelGGL((kq_paged_merge_kernel<D, BF>), dim3((unsigned)(((int64_t)a.T * a.Hq + 3) / 4)), dim3(256), 0,
                           s, a);
}

// Partial slots of a call: a row's n * Hq * splits is below (kSplitWaves + waves)
// * 16 for waves < kSplitWaves (with as many or more it is not split), and no
// row has more splits than one token over max_kv keys.
int64_t max_slots(int64_t T, int64_t B, int Hq, int Hkv, int max_kv) {
    const int most = paged_splits(1, max_kv, Hq / Hkv, Hkv);
    if (most < 2) return 0;
    const int64_t by_token = T * Hq * most, by_row = B * 2 * kSplitWaves * 16;
    return by_token < by_row ? by_token : by_row;
}

size_t part_bytes(int64_t slots, int D) { return ((size_t)slots * D * 4 + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

size_t kq_sdpa_paged_workspace_bytes(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q,
                                     int32_t max_kv, int q8) {
    if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || max_q <= 0 || max_kv <= 0) return 0;
    const int64_t slots = max_slots(T, B, Hq, Hkv, max_kv);
    return slots ? part_bytes(slots, D) + (size_t)slots * 8 : 0;
}

int kq_sdpa_paged(const void *q, int64_t q_stride, const kq_paged_pool *pool, const int32_t *block_table,
                  int64_t table_stride, int32_t table_width, const int32_t *kv_lens, const int32_t *cu_q, int32_t T,
                  int32_t B, int32_t Hq, int32_t max_q, int32_t max_kv, float scale, void *out, int64_t out_stride,
                  void *workspace, size_t workspace_bytes, kq_stream_t stream) {
    if (const int rc = kq_pool_check(pool)) return rc;
    if (T == 0 || B == 0) return KQ_OK;
    if (!q || !block_table || !kv_lens || !cu_q || !out) return KQ_ERR_NULL_POINTER;
    const int Hkv = pool->Hkv, D = pool->D;
    if (T < 0 || B < 0 || B > (1 << 20) || Hq <= 0 || Hq % Hkv || Hq / Hkv > 64 || max_q < 1 || max_kv < 1 ||
        table_width < 1 || table_stride < table_width)
        return KQ_ERR_BAD_SHAPE;
    if ((int64_t)T * Hq > (1 << 30) || q_stride < (int64_t)Hq * D || out_stride < (int64_t)Hq * D)
        return KQ_ERR_BAD_SHAPE;
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_stride | out_stride) & 7)) return KQ_ERR_BAD_ALIGN;
    const size_t need = kq_sdpa_paged_workspace_bytes(T, B, Hq, Hkv, D, max_q, max_kv, pool->k_scales != nullptr);
    if (need && (!workspace || workspace_bytes < need)) return KQ_ERR_WORKSPACE_TOO_SMALL;
    if (need && ((uintptr_t)workspace & 255)) return KQ_ERR_BAD_ALIGN;
    PagedArgs a;
    a.q = (const uint16_t *)q;
    a.out = (uint16_t *)out;
    a.k = pool->k;
    a.v = pool->v;
    a.ks = (const uint16_t *)pool->k_scales;
    a.kb = (const uint16_t *)pool->k_biases;
    a.vs = (const uint16_t *)pool->v_scales;
    a.vb = (const uint16_t *)pool->v_biases;
    a.table = block_table;
    a.kv_lens = kv_lens;
    a.cu_q = cu_q;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.page_stride = pool->page_stride;
    a.head_stride = pool->head_stride;
    a.table_stride = table_stride;
    a.tok_stride = (int32_t)pool->token_stride;
    a.lps = __builtin_ctz(pool->page_size);
    a.n_pages = pool->n_pages;
    a.width = table_width;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.scale_log2 = scale * 1.4426950408889634f;
    const int64_t slots = max_slots(T, B, Hq, Hkv, max_kv);
    a.part = (float *)workspace;
    a.ml = (float *)((char *)workspace + part_bytes(slots, D));
    // units of the longest rows; the grid's waves take the rest in turn
    const int64_t blocks = ((int64_t)T * a.G + 15) / 16 + B;
    const int64_t units = blocks * Hkv * paged_splits(1, max_kv, a.G, Hkv);
    const int grid = (int)(units < (1 << 16) ? units : (1 << 16));
    const bool q8 = a.ks != nullptr, bf = pool->dtype == KQ_DTYPE_BF16;
    hipStream_t s = (hipStream_t)stream;
    const bool merge = slots > 0;
    switch (D) {
    case 64: bf ? launch<64, true>(a, q8, grid, merge, s) : launch<64, false>(a, q8, grid, merge, s); break;
    case 96: bf ? launch<96, true>(a, q8, grid, merge, s) : launch<96, false>(a, q8, grid, merge, s); break;
    case 128: bf ? launch<128, true>(a, q8, grid, merge, s) : launch<128, false>(a, q8, grid, merge, s); break;
    case 256: bf ? launch<256, true>(a, q8, grid, merge, s) : launch<256, false>(a, q8, grid, merge, s); break;
    default: bf ? launch<512, true>(a, q8, grid, merge, s) : launch<512, false>(a, q8, grid, merge, s); break;
    }
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

}  // extern "C"
