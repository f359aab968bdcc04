// Queries and keys normed for each head and rotated by their positions
// (kq_rope_qk), the keys and the values beside them going straight to a paged
// cache's slots in the second form (kq_paged_write_rope).
//
// A head's row x of D values, normed where there is a weight w:
//   y = x * w / sqrt(mean(x^2) + eps)
// and its first R values turned in pairs (a, b), at position p with f radians a
// position:
//   a' = (a cos(p f) - b sin(p f)) factor,  b' = (b cos(p f) + a sin(p f)) factor,
// pair j being y[j], y[j + R / 2], or with `interleaved` y[2 j], y[2 j + 1].  All
// in fp32, rounded once; p f in 64 bits, of which the whole turns are taken off
// before the 32-bit sine: a position of 10^6 in fp32 would be off by 0.03 radians.
#include <algorithm>

#include "kq_paged_store.h"

namespace {

struct RopeArgs {
    const uint16_t *src[3];  // q, k, v
    uint16_t *dst[2];        // q, k (k not where the cache takes it)
    int64_t token_stride[3], head_stride[3], out_token_stride[2], out_head_stride[2];
    const int32_t *positions, *slots;
    const double *freqs;
    const void *weight[2];
    kq_paged_pool pool;
    float eps, factor;
    int32_t T, Hq, Hkv, rows;  // rows: heads of q, k and, where they are stored, v
    int32_t R, interleaved, weight_f32, lps;
    int32_t tokens;  // of a workgroup that takes several
};

// The most tokens of a workgroup: 8 KB of sines and cosines.
constexpr int most_tokens(int D) { return 2048 / D; }

template <bool BF>
__device__ __forceinline__ void unpack8(const u32x4 &v, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f16bits_to_f32<BF>((v[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
}

// Sum over the LG lanes of a head's row, in all of them: row operations inside the
// VALU up to 16 lanes, swaps of rows and halves past them.
template <int CTRL>
__device__ __forceinline__ float add_lane(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int LG>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (LG == 8) {
        v = add_lane<0xB1>(v);   // neighbours, pairs, then halves of eight (mirrored)
        v = add_lane<0x4E>(v);
        return add_lane<0x141>(v);
    }
    v = add_lane<0x128>(v);  // row_ror:8, 4, 2, 1
    v = add_lane<0x124>(v);
    v = add_lane<0x122>(v);
    v = add_lane<0x121>(v);
    if constexpr (LG >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto w = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (uint32_t)w[0]) + __builtin_bit_cast(float, (uint32_t)w[1]);
    }
    if constexpr (LG == 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (uint32_t)w[0]) + __builtin_bit_cast(float, (uint32_t)w[1]);
    }
    return v;
}

// A workgroup takes PASSES times 256 / LG heads' rows of one token, LG lanes a
// row and 8 values a lane.  The token's sines and cosines are made once, a pair a
// thread, and shared through LDS, and so are the weights (loaded where they are
// used, behind the barrier, 8192 tokens took 40.5 us in place of 35.6).  A lane loads its pairs' other halves itself,
// from the lines that its row's lanes have just asked for.  Rows are loaded before
// any is stored, by the same wave, so outputs may be the inputs.  MANY: a.tokens
// tokens of few heads share a workgroup (66425 tokens of 2 + 1 heads of 64 83 us
// with one each, 21 so).
template <int D, bool BF, bool Q8, bool WRITE, int PASSES, bool MANY>
__global__ __launch_bounds__(256) void kq_rope_kernel(RopeArgs a) {
    constexpr int L = D / 8, LG = L <= 8 ? 8 : L <= 16 ? 16 : L <= 32 ? 32 : 64, RP = 256 / LG;
    constexpr int TOKENS = MANY ? most_tokens(D) : 1;
    __shared__ __attribute__((aligned(16))) float cs[TOKENS * (D / 2)], sn[TOKENS * (D / 2)], weight[2][D];
    const int t0 = MANY ? blockIdx.x * a.tokens : blockIdx.x;
    const int tokens = MANY ? min(a.tokens, a.T - t0) : 1;
    if (!MANY && a.positions[t0] < 0) return;
    const int c = threadIdx.x % LG, row0 = blockIdx.y * (RP * PASSES) + threadIdx.x / LG;
    const int half = a.R / 2;
    // where this lane's pairs' other halves lie: in itself, or half the rotated part away
    const bool turned = 8 * c < a.R, apart = turned && !a.interleaved, low = 8 * c < half;
    const int other = !apart ? c : low ? c + half / 8 : c - half / 8;
    u32x4 v[PASSES], vo[PASSES];
    int which[PASSES], head[PASSES], at[PASSES];  // at: the token's number in the workgroup, -1: no row
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int item = row0 + p * RP, nth = MANY ? item / a.rows : 0, row = item - nth * a.rows;
        const int t = t0 + nth;
        at[p] = !MANY || (nth < tokens && a.positions[t] >= 0) ? nth : -1;
        which[p] = row < a.Hq ? 0 : row < a.Hq + a.Hkv ? 1 : 2;
        head[p] = row - (which[p] == 0 ? 0 : which[p] == 1 ? a.Hq : a.Hq + a.Hkv);
        v[p] = vo[p] = u32x4{0u, 0u, 0u, 0u};
        if ((MANY ? at[p] >= 0 : row < a.rows) && c < L) {
            const uint16_t *x = which[p] == 0   ? a.src[0] + t * a.token_stride[0] + head[p] * a.head_stride[0]
                                : which[p] == 1 ? a.src[1] + t * a.token_stride[1] + head[p] * a.head_stride[1]
                                                : a.src[2] + t * a.token_stride[2] + head[p] * a.head_stride[2];
            v[p] = *(const u32x4 *)(x + 8 * c);
            if (which[p] < 2 && apart) vo[p] = *(const u32x4 *)(x + 8 * other);
        }
    }
#pragma unroll
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
        const int d = i % D;
        if (const void *w = i < D ? a.weight[0] : a.weight[1])
            weight[i / D][d] = a.weight_f32 ? ((const float *)w)[d] : f16bits_to_f32<BF>(((const uint16_t *)w)[d]);
    }
    for (int i = threadIdx.x; i < tokens * half; i += 256) {
        const int nth = MANY ? i / half : 0;
        const double turns = (double)a.positions[t0 + nth] * a.freqs[i - nth * half] * 0.15915494309189533577;
        float s, co;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &co);
        cs[i] = co * a.factor;
        sn[i] = s * a.factor;
    }
    __syncthreads();
    // a value becomes itself times its cosine plus its pair's other times +-its sine
    float co[8], si[8];
    const auto turn = [&](int nth) {
        if (!turned) return;
        const int j = nth * half + (a.interleaved ? 4 * c : low ? 8 * c : 8 * c - half);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = j + (a.interleaved ? i / 2 : i);
            co[i] = cs[k];
            si[i] = (a.interleaved ? i % 2 == 0 : low) ? -sn[k] : sn[k];
        }
    };
    if constexpr (!MANY) turn(0);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        // (uniform over a row's lanes, as all below is)
        if constexpr (MANY) {
            if (at[p] < 0) continue;
        } else {
            if (row0 + p * RP >= a.rows) break;
        }
        const int t = t0 + at[p];
        if constexpr (MANY) turn(at[p]);
        u32x4 out = v[p];
        if (which[p] < 2) {
            float x[8], xo[8];
            unpack8<BF>(v[p], x);
            unpack8<BF>(vo[p], xo);
            if (which[p] == 0 ? a.weight[0] : a.weight[1]) {
                const float *wx = weight[which[p]] + 8 * min(c, L - 1), *wo = weight[which[p]] + 8 * min(other, L - 1);
                const auto mean = [&](float eps) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
                    return fmaf(row_sum<LG>(sum), 1.f / D, eps);
                };
                float m = mean(a.eps);
                if (BF && !(m >= 0x1p-100f && m <= 3.4028235e38f)) {
                    // squares past the ends of fp32: of the values times a power of two
                    const float by = m < 1.f ? 0x1p70f : 0x1p-70f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] *= by;
                        xo[i] *= by;
                    }
                    m = mean(a.eps * by * by);
                }
                const float inv = rsqrtf(m);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = x[i] * inv * wx[i];
                    xo[i] = xo[i] * inv * wo[i];
                }
            }
            if (turned) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = fmaf(x[i], co[i], (a.interleaved ? x[i ^ 1] : xo[i]) * si[i]);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = pack2<BF>(x[2 * i], x[2 * i + 1]);
        }
        if (!WRITE || which[p] == 0) {
            if (c < L) {
                uint16_t *y = which[p] == 0 ? a.dst[0] + t * a.out_token_stride[0] + head[p] * a.out_head_stride[0]
                                            : a.dst[1] + t * a.out_token_stride[1] + head[p] * a.out_head_stride[1];
                *(u32x4 *)(y + 8 * c) = out;
            }
        } else {
            const int64_t to = slot_offset(a.pool, a.lps, a.slots[t], head[p]);
            if (to >= 0 && c < L) store_values<BF, Q8>(a.pool, which[p] - 1, to, c, out);
        }
    }
}

template <int D, bool BF, bool Q8, bool WRITE>
void launch(RopeArgs a, hipStream_t s) {
    constexpr int L = D / 8, LG = L <= 8 ? 8 : L <= 16 ? 16 : L <= 32 ? 32 : 64, RP = 256 / LG;
    const int groups = (a.rows + RP - 1) / RP, groups3 = (a.rows + 3 * RP - 1) / (3 * RP);
    // Three passes where one would give the GPU four workgroups a CU (us with 1 / 2 / 3
    // passes, 32 + 8 heads of 128: 33 tokens 4.9 / 5.0 / 5.1, 128 4.8 / 5.1 / 5.2, 512 5.7 /
    // 5.7 / 5.8, 1024 9.1 / 7.8 / 8.0, 2048 14.1 / 13.4 / 12.9, 8192 45.5 / 42.3 / 35.6; a
    // copy of 2048 tokens' bytes 7.6, of 8192 33.7).  Three tokens or more a workgroup
    // where they fit these passes and leave 1024 workgroups (one / several, 20000
    // tokens of 4 + 1 heads of 128 36 / 20, 10000 of 8 + 1 22 / 16; but two each, 4097 of 16
    // + 4 14.1 / 15.0, and 1100 of 4 + 4 of 64, which 92 would take, 5.4 / 5.9).
    if ((int64_t)a.T * groups < 1024) {
        hipLaunchKernelGGL((kq_rope_kernel<D, BF, Q8, WRITE, 1, false>), dim3(a.T, groups), dim3(256), 0, s, a);
        return;
    }
    a.tokens = std::min({3 * RP / a.rows, most_tokens(D), a.T / 1024});
    if (a.tokens > 2)
        hipLaunchKernelGGL((kq_rope_kernel<D, BF, Q8, WRITE, 3, true>), dim3((a.T + a.tokens - 1) / a.tokens), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((kq_rope_kernel<D, BF, Q8, WRITE, 3, false>), dim3(a.T, groups3), dim3(256), 0, s, a);
}

template <int D, bool BF>
void launch_form(const RopeArgs &a, bool write, bool q8, hipStream_t s) {
    if (!write) return launch<D, BF, false, false>(a, s);
    if constexpr (D % 64 == 0)
        if (q8) return launch<D, BF, true, true>(a, s);
    launch<D, BF, false, true>(a, s);
}

int launch_all(const RopeArgs &a, int D, int dtype, bool write, bool q8, hipStream_t s) {
    const bool bf = dtype == KQ_DTYPE_BF16;
    switch (D) {
    case 64: bf ? launch_form<64, true>(a, write, q8, s) : launch_form<64, false>(a, write, q8, s); break;
    case 96: bf ? launch_form<96, true>(a, write, q8, s) : launch_form<96, false>(a, write, q8, s); break;
    case 128: bf ? launch_form<128, true>(a, write, q8, s) : launch_form<128, false>(a, write, q8, s); break;
    case 256: bf ? launch_form<256, true>(a, write, q8, s) : launch_form<256, false>(a, write, q8, s); break;
    default: bf ? launch_form<512, true>(a, write, q8, s) : launch_form<512, false>(a, write, q8, s); break;
    }
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

// What both forms share of a call; T > 0.
int fill(RopeArgs &a, const kq_rope *r, const int32_t *positions, int32_t T, int D, int dtype, const kq_rope_rows *q,
         const kq_rope_rows *k) {
    if (!r || !r->freqs || !positions || !q || !k) return KQ_ERR_NULL_POINTER;
    if (dtype != KQ_DTYPE_F16 && dtype != KQ_DTYPE_BF16) return KQ_ERR_UNSUPPORTED_DTYPE;
    if (D != 64 && D != 96 && D != 128 && D != 256 && D != 512) return KQ_ERR_BAD_SHAPE;
    // (a grid of fewer than 2^32 threads)
    if (T < 0 || T > 1 << 23 || r->rotary_dim < 16 || r->rotary_dim > D || r->rotary_dim % 16) return KQ_ERR_BAD_SHAPE;
    if (q->heads < 0 || k->heads < 0 || q->heads > 1 << 16 || k->heads > 1 << 16) return KQ_ERR_BAD_SHAPE;
    if (r->weight_dtype != dtype && r->weight_dtype != KQ_DTYPE_F32 && (r->q_weight || r->k_weight))
        return KQ_ERR_UNSUPPORTED_DTYPE;
    // (of a NaN neither holds)
    if (!(r->eps >= 0.f && r->eps <= 3.4028235e38f) || !(fabsf(r->factor) <= 3.4028235e38f)) return KQ_ERR_BAD_ARGUMENT;
    if (((uintptr_t)r->freqs & 7) || (((uintptr_t)r->q_weight | (uintptr_t)r->k_weight) & 15)) return KQ_ERR_BAD_ALIGN;
    const kq_rope_rows *rows[2] = {q, k};
    for (int i = 0; i < 2; ++i) {
        a.src[i] = (const uint16_t *)rows[i]->x;
        a.token_stride[i] = rows[i]->token_stride;
        a.head_stride[i] = rows[i]->head_stride;
        a.dst[i] = (uint16_t *)rows[i]->out;
        a.out_token_stride[i] = rows[i]->out_token_stride;
        a.out_head_stride[i] = rows[i]->out_head_stride;
        if (rows[i]->heads && !a.src[i]) return KQ_ERR_NULL_POINTER;
        if ((((uintptr_t)a.src[i] | (uintptr_t)a.dst[i]) & 15) ||
            ((a.token_stride[i] | a.head_stride[i] | a.out_token_stride[i] | a.out_head_stride[i]) & 7))
            return KQ_ERR_BAD_ALIGN;
    }
    a.positions = positions;
    a.freqs = r->freqs;
    a.weight[0] = r->q_weight;
    a.weight[1] = r->k_weight;
    a.weight_f32 = r->weight_dtype == KQ_DTYPE_F32;
    a.eps = r->eps;
    a.factor = r->factor;
    a.R = r->rotary_dim;
    a.interleaved = r->interleaved;
    a.T = T;
    a.Hq = q->heads;
    a.Hkv = k->heads;
    a.rows = q->heads + k->heads;
    return KQ_OK;
}

}  // namespace

extern "C" {

int kq_rope_qk(const kq_rope *rope, const int32_t *positions, int32_t T, int32_t D, int dtype, const kq_rope_rows *q,
               const kq_rope_rows *k, kq_stream_t stream) {
    if (T == 0) return KQ_OK;
    RopeArgs a{};
    if (const int rc = fill(a, rope, positions, T, D, dtype, q, k)) return rc;
    if ((a.Hq && !a.dst[0]) || (a.Hkv && !a.dst[1])) return KQ_ERR_NULL_POINTER;
    if (!a.rows) return KQ_OK;
    return launch_all(a, D, dtype, false, false, (hipStream_t)stream);
}

int kq_paged_write_rope(const kq_paged_pool *pool, const kq_rope *rope, const int32_t *positions, const int32_t *slots,
                        int32_t T, const kq_rope_rows *q, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                        const void *v, int64_t v_token_stride, int64_t v_head_stride, kq_stream_t stream) {
    if (const int rc = kq_pool_check(pool)) return rc;
    if (T == 0) return KQ_OK;
    if (!k || !v || !slots) return KQ_ERR_NULL_POINTER;
    const kq_rope_rows keys{k, nullptr, k_token_stride, k_head_stride, 0, 0, pool->Hkv};
    RopeArgs a{};
    if (const int rc = fill(a, rope, positions, T, pool->D, pool->dtype, q, &keys)) return rc;
    if (a.Hq && !a.dst[0]) return KQ_ERR_NULL_POINTER;
    if (!kq_pool_places_apart(*pool)) return KQ_ERR_BAD_ARGUMENT;
    if (((uintptr_t)v & 15) || ((v_token_stride | v_head_stride) & 7)) return KQ_ERR_BAD_ALIGN;
    a.src[2] = (const uint16_t *)v;
    a.token_stride[2] = v_token_stride;
    a.head_stride[2] = v_head_stride;
    a.slots = slots;
    a.pool = *pool;
    a.lps = __builtin_ctz(pool->page_size);
    a.rows += pool->Hkv;
    return launch_all(a, pool->D, pool->dtype, true, pool->k_scales != nullptr, (hipStream_t)stream);
}

}  // extern "C"
