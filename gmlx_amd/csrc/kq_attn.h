// Helpers that the decode and the paged attention kernels share: MFMA and
// 16-bit conversions by element type, reductions over a wave's lane groups.
#pragma once
#include <stdlib.h>

#include <initializer_list>
#include <type_traits>

#include "kq_common.h"

int device_cus();

namespace {

template <bool BF>
__device__ __forceinline__ floatx4 mfma(const half8_t &a, const half8_t &b, const floatx4 &c) {
    if constexpr (!BF) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    } else {
        typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (!BF) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
    } else {
        return kq_f32x2_to_bf16_bits(a, b);
    }
}

template <bool BF>
__device__ __forceinline__ uint16_t from_f32(float f) {
    if constexpr (!BF) return __builtin_bit_cast(uint16_t, (_Float16)f);
    else return kq_f32_to_bf16_bits(f);
}

// Largest of v over the four lane groups (lanes r, r + 16, r + 32, r + 48), in
// every one of them: row swaps inside the VALU, where LDS shuffles put two
// round trips into a tile's serial chain.
__device__ __forceinline__ float max_over_groups(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __builtin_bit_cast(
        uint32_t, fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// 16-bit float bits (fp16, or bf16 when BF) -> fp32
template <bool BF>
__device__ __forceinline__ float f16bits_to_f32(uint32_t h) {
    if constexpr (BF) return __builtin_bit_cast(float, h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// A wave-uniform value the compiler cannot prove uniform, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// Tokens per split of a row, by the row's own length.
struct SplitRule {
    int32_t one, to64, to128, to256, rest;

    __host__ __device__ __forceinline__ int tokens(int len) const {
        return len <= one ? one : len <= to64 ? 64 : len <= to128 ? 128 : len <= to256 ? 256 : rest;
    }
};

// Split lengths of decode rows, over contiguous caches and pages alike: short rows
// one split, then 64, 128 and 256 tokens up to the lines, past them 512 (measured
// beside split_rule in kq_attention.hip and wave_rule in kq_paged.hip).
SplitRule row_split_rule(int Hq, int Hkv, int D, bool q8) {
    if (D > 128) return SplitRule{q8 || D > 256 ? 0 : 128, 1024, 8192, 32768, 512};
    if (q8) return SplitRule{Hq > 8 * Hkv ? 256 : 0, 1024, 2048, 32768, 512};
    if (Hq > 8 * Hkv) return SplitRule{512, 0, 1024, 8192, 512};
    return SplitRule{256, 512, Hq > 4 * Hkv ? 1024 : 4096, 8192, 512};
}

__host__ __device__ __forceinline__ int row_splits(const SplitRule &rule, int len) {
    const int split = rule.tokens(len);
    return len <= 0 ? 1 : (len + split - 1) / split;
}

// The most splits of any row of at most max_len keys: those of max_len or of a
// row at a line below it.
int most_row_splits(const SplitRule &rule, int max_len) {
    int most = row_splits(rule, max_len);
    for (const int line : {rule.one, rule.to64, rule.to128, rule.to256}) {
        const int n = line < max_len ? row_splits(rule, line) : 1;
        if (n > most) most = n;
    }
    return most;
}

int env_int(const char *name, int dflt) {
    const char *s = getenv(name);
    if (!s || !*s) return dflt;
    char *end = nullptr;
    const long v = strtol(s, &end, 10);
    return (end && *end == 0 && v > 0 && v < (1 << 24)) ? (int)v : dflt;
}

}  // namespace
