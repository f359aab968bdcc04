// Where a token's row lies in the paged cache's pool, and how 8 values of it are
// stored there, for the kernels that write the pool.
#pragma once
#include "kq_paged.h"

namespace {

// Element (byte, 8-bit pool) offset of a slot's row of head h; -1 outside the pool.
__device__ __forceinline__ int64_t slot_offset(const kq_paged_pool &p, int lps, int slot, int h) {
    const int page = slot >> lps;
    if (slot < 0 || page >= p.n_pages) return -1;
    return page * p.page_stride + h * p.head_stride + (slot & ((1 << lps) - 1)) * p.token_stride;
}

// Smallest, largest and sum of what a group's 8 threads hold.
__device__ __forceinline__ void group_range(float &lo, float &hi, float &odd) {
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, off));
        hi = fmaxf(hi, __shfl_xor(hi, off));
        odd += __shfl_xor(odd, off);
    }
}

// Values 8 c .. 8 c + 7 (w: 16-bit) of a row to the place `to` of the pool's K (kv
// 0) or V; the 8 lanes of a 64-value group call it together.
template <bool BF, bool Q8>
__device__ __forceinline__ void store_values(const kq_paged_pool &p, int kv, int64_t to, uint32_t c, const u32x4 &w) {
    if constexpr (!Q8) {
        *(u32x4 *)((uint16_t *)(kv ? p.v : p.k) + to + 8 * c) = w;
    } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = f16bits_to_f32<BF>(w[i] & 0xFFFFu);
            x[2 * i + 1] = f16bits_to_f32<BF>(w[i] >> 16);
        }
        float lo = x[0], hi = x[0], odd = x[0] - x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
            odd += x[i] - x[i];  // NaN from an infinity or NaN (which fminf drops), else 0
        }
        group_range(lo, hi, odd);
        // (bf16 values can be further apart than fp32's largest: halves of all then)
        const float part = BF && !(hi - lo <= 3.4028235e38f) ? 0.5f : 1.f;
        // the scale as it is stored: the values are rounded against what is
        // read back; a bias of 16 bits holds lo exactly
        const uint16_t s16 = from_f32<BF>((hi * part - lo * part) / (255.f * part) + odd);
        const float s = f16bits_to_f32<BF>(s16);
        uint32_t q[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = s == 0.f ? 0.f : fminf(fmaxf(rintf((x[i] * part - lo * part) / (s * part)), 0.f), 255.f);
            q[i >> 2] |= (uint32_t)v << (8 * (i & 3));
        }
        *(u32x2 *)((uint8_t *)(kv ? p.v : p.k) + to + 8 * c) = u32x2{q[0], q[1]};
        if ((c & 7) == 0) {
            const int64_t g = (to + 8 * c) >> 6;
            ((uint16_t *)(kv ? p.v_scales : p.k_scales))[g] = s16;
            ((uint16_t *)(kv ? p.v_biases : p.k_biases))[g] = from_f32<BF>(lo);
        }
    }
}

}  // namespace
