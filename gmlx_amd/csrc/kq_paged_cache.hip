// The paged KV cache's bookkeeping and copies (kq_capi.h): kq_paged_plan,
// kq_paged_write, kq_paged_read.
#include <algorithm>

#include "kq_paged.h"
#include "kq_paged_store.h"

int kq_pool_check(const kq_paged_pool *p) {
    if (!p || !p->k || !p->v) return KQ_ERR_NULL_POINTER;
    if (p->dtype != KQ_DTYPE_F16 && p->dtype != KQ_DTYPE_BF16) return KQ_ERR_UNSUPPORTED_DTYPE;
    const int D = p->D, ps = p->page_size;
    if (D != 64 && D != 96 && D != 128 && D != 256 && D != 512) return KQ_ERR_BAD_SHAPE;
    if (p->n_pages < 1 || p->Hkv < 1 || p->Hkv > 1024 || ps < 16 || ps > 1024 || (ps & (ps - 1)))
        return KQ_ERR_BAD_SHAPE;
    if ((int64_t)p->n_pages * ps >= (int64_t)1 << 31) return KQ_ERR_BAD_SHAPE;
    const bool q8 = p->k_scales || p->k_biases || p->v_scales || p->v_biases;
    if (q8 && (!p->k_scales || !p->k_biases || !p->v_scales || !p->v_biases)) return KQ_ERR_NULL_POINTER;
    // 32-bit offsets within a page
    if (p->token_stride < D || p->token_stride > (1 << 20) || p->head_stride < 0 || p->page_stride < 0)
        return KQ_ERR_BAD_SHAPE;
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return KQ_ERR_BAD_ALIGN;
    const int64_t al = q8 ? 63 : 7;
    if ((p->page_stride | p->head_stride | p->token_stride) & al) return KQ_ERR_BAD_ALIGN;
    if (q8) {
        if (D == 96 || p->token_stride != D) return KQ_ERR_BAD_SHAPE;
        if (((uintptr_t)p->k_scales | (uintptr_t)p->k_biases | (uintptr_t)p->v_scales | (uintptr_t)p->v_biases) & 1)
            return KQ_ERR_BAD_ALIGN;
    }
    return KQ_OK;
}

// Whether no two places of K and V lie on the same memory as far as the strides
// and bases tell: each stride passes what the smaller ones reach (a page or head
// that is repeated by a stride of 0 does not), and K is not V.  Rows written to
// such places by different threads would be mixed.
bool kq_pool_places_apart(const kq_paged_pool &p) {
    struct { int64_t stride, n; } d[3] = {{p.token_stride, p.page_size}, {p.head_stride, p.Hkv}, {p.page_stride, p.n_pages}};
    std::sort(d, d + 3, [](const auto &x, const auto &y) { return x.stride < y.stride; });
    __int128 reach = p.D;
    for (const auto &x : d) {
        if (x.n == 1) continue;
        if (x.stride < reach) return false;
        reach += (__int128)x.stride * (x.n - 1);
    }
    const void *at[4] = {p.k_scales, p.k_biases, p.v_scales, p.v_biases};
    for (int i = 0; p.k_scales && i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (at[i] == at[j]) return false;
    return p.k != p.v;
}

namespace {

// ---- the plan ------------------------------------------------------------
// With P = page_size and the row's base = min(keep, seq):
//   have = ceil(seq / P), want = ceil((base + new) / P),
//   give = max(have - want, 0), take = max(want - have, 0),
// the stack with the released pages on it is S[i] = free[i] (i < count), then
// the rows' table entries want .. have in row order; total = count + sum of
// give; page j that row b takes is S[total - 1 - (sum of take before b) - j].
// Everything follows from three exclusive sums over the rows, which each
// workgroup makes for itself in LDS (2048 rows: two a thread), so one launch
// with no exchange between workgroups does it all; tokens, taken and returned
// pages are then spread over the grid, each finding its row by binary search.
// Bound by its chain of dependent loads, barriers and searches: 8 rows 4.6 us,
// 300 rows with 2048 tokens 7.1 (138 KB read and written).
struct PlanArgs {
    const int32_t *seq, *keep, *add, *count;
    int32_t *table, *stack, *cu, *kv, *slots, *pos, *count_out, *refused;
    int64_t table_stride;
    int32_t B, width, n_stack, lps, max_tokens;
};

constexpr int kPlanThreads = 1024;

struct PlanRows {
    int cu[KQ_PAGED_MAX_ROWS + 1];    // new tokens before row b
    int take[KQ_PAGED_MAX_ROWS + 1];  // pages taken before row b
    int give[KQ_PAGED_MAX_ROWS + 1];  // pages released before row b
    int base[KQ_PAGED_MAX_ROWS];      // kept tokens, -1: refused
    int pages[KQ_PAGED_MAX_ROWS];     // have (rows that take), want (rows that give)
};

// Exclusive sum of v over the workgroup's threads; total in every thread.
__device__ __forceinline__ int block_sum(int v, int *wave, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int inc = v;
    for (int off = 1; off < 64; off <<= 1) {
        const int t = __shfl_up(inc, off);
        if (lane >= off) inc += t;
    }
    __syncthreads();  // the last sum's reads
    if (lane == 63) wave[w] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        const int t = wave[i];
        if (i < w) before += t;
        total += t;
    }
    return before + inc - v;
}

// The last row whose first item is at or before i (rows without items are
// passed over, as the next row starts where they do).
__device__ __forceinline__ int row_of(const int *first, int B, int i) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void kq_paged_plan_kernel(PlanArgs a) {
    __shared__ PlanRows r;
    __shared__ int wave[kPlanThreads / 64];
    __shared__ int taken;  // pages that the served rows take
    constexpr int PER = KQ_PAGED_MAX_ROWS / kPlanThreads;
    const int t = threadIdx.x, P = 1 << a.lps;
    if (t == 0) taken = 0;
    int seq[PER], base[PER], add[PER], have[PER], want[PER], give[PER], take[PER];
    int s_add = 0, s_give = 0, s_take = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = t * PER + i;
        const bool in = b < a.B;
        seq[i] = in ? (int)min((int64_t)max(a.seq[b], 0), (int64_t)a.width << a.lps) : 0;
        base[i] = in && a.keep ? min(max(a.keep[b], 0), seq[i]) : seq[i];
        add[i] = in ? max(a.add[b], 0) : 0;
        have[i] = (seq[i] + P - 1) >> a.lps;
        want[i] = (int)(((int64_t)base[i] + add[i] + P - 1) >> a.lps);
        const bool fits = want[i] <= a.width;
        give[i] = max(have[i] - want[i], 0);
        take[i] = fits ? max(want[i] - have[i], 0) : 0;
        if (!fits) base[i] = -1;
        s_add += add[i];
        s_give += give[i];
        s_take += take[i];
    }
    int n_add, n_give, n_take;
    int e_add = block_sum(s_add, wave, n_add);
    int e_give = block_sum(s_give, wave, n_give);
    int e_take = block_sum(s_take, wave, n_take);
    const int count = min(max(a.count[0], 0), a.n_stack);
    const int total = min(count + n_give, a.n_stack);
    int served = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = t * PER + i;
        if (take[i] > 0) {
            if (e_take + take[i] <= total) served = e_take + take[i];
            else base[i] = -1;
        }
        if (b <= a.B) {
            r.cu[b] = e_add;
            r.take[b] = e_take;
            r.give[b] = e_give;
        }
        if (b < a.B) {
            r.base[b] = base[i];
            r.pages[b] = give[i] > 0 ? want[i] : have[i];
            if (blockIdx.x == 0) {
                a.cu[b] = e_add;
                a.kv[b] = base[i] < 0 ? seq[i] : base[i] + add[i];
                a.refused[b] = base[i] < 0;
            }
        }
        e_add += add[i];
        e_give += give[i];
        e_take += take[i];
    }
    if (t == 0) {
        // (2048 rows fill every thread's share: nobody holds b == B)
        r.cu[a.B] = n_add;
        r.take[a.B] = n_take;
        r.give[a.B] = n_give;
    }
    if (served) atomicMax(&taken, served);
    __syncthreads();
    const int used = taken, left = total - used;
    if (blockIdx.x == 0 && t == 0) {
        a.cu[a.B] = n_add;
        a.count_out[0] = left;
    }
    // S[i]
    auto stack = [&](int i) {
        if (i < count) return a.stack[i];
        const int b = row_of(r.give, a.B, i - count);
        return a.table[b * a.table_stride + r.pages[b] + (i - count - r.give[b])];
    };
    const int step = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + t;
    for (int i = first; i < a.max_tokens; i += step) {
        int slot = -1, p = -1;
        if (i < n_add) {
            const int b = row_of(r.cu, a.B, i);
            if (r.base[b] >= 0) {
                p = (int)((uint32_t)r.base[b] + (uint32_t)i - (uint32_t)r.cu[b]);
                const int nth = p >> a.lps, fresh = nth - r.pages[b], from = total - 1 - (r.take[b] + fresh);
                // (a row that gives pages has want in r.pages, past its last token;
                // p and from are only negative where new_lens add up past 31 bits)
                const int page = p < 0 || (fresh >= 0 && from < 0) ? -1
                                 : fresh < 0 ? a.table[b * a.table_stride + nth] : stack(from);
                slot = page < 0 || page >= (0x7fffffff >> a.lps) ? -1 : (page << a.lps) + (p & (P - 1));
            }
        }
        a.slots[i] = slot;
        a.pos[i] = p;
    }
    for (int i = first; i < used; i += step) {
        const int b = row_of(r.take, a.B, i);
        a.table[b * a.table_stride + r.pages[b] + (i - r.take[b])] = stack(total - 1 - i);
    }
    for (int i = count + first; i < left; i += step) a.stack[i] = stack(i);
}

// ---- write and read --------------------------------------------------------
// A thread moves 8 values (16 bytes of a 16-bit row); L = D / 8 threads a row
// of a head, blockIdx.y K or V.  HBM-bound where rows are many: 4097 tokens of 8
// heads, head dim 128 (33.6 MB each way a call), written in 7.6 us and read in 7.5,
// 4.4 TB/s; 32 tokens 2.7 (the launch).  2048 tokens (12.7 MB) to 8 bits 7.1, by
// vector issue: 306 instructions a wave, about 85 of them the nine exact divisions,
// fill 91 % of the busy cycles; back 5.2, its loads' latency in one round of waves.
struct CopyArgs {
    kq_paged_pool p;
    const uint16_t *src[2];
    uint16_t *dst[2];
    int64_t token_stride[2], head_stride[2];
    const int32_t *slots;
    int32_t T, lps;
    uint32_t rows;  // T * Hkv
};

template <int D, bool BF, bool Q8>
__global__ __launch_bounds__(256) void kq_paged_write_kernel(CopyArgs a) {
    constexpr int L = D / 8;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x, row = item / L, c = item - row * L;
    if (row >= a.rows) return;
    const int kv = blockIdx.y;
    const uint32_t t = row / (uint32_t)a.p.Hkv, h = row - t * a.p.Hkv;
    const int64_t to = slot_offset(a.p, a.lps, a.slots[t], h);
    if (to < 0) return;  // uniform over a row's threads
    const u32x4 w = *(const u32x4 *)(a.src[kv] + t * a.token_stride[kv] + h * a.head_stride[kv] + 8 * c);
    store_values<BF, Q8>(a.p, kv, to, c, w);
}

template <int D, bool BF, bool Q8>
__global__ __launch_bounds__(256) void kq_paged_read_kernel(CopyArgs a) {
    constexpr int L = D / 8;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x, row = item / L, c = item - row * L;
    if (row >= a.rows) return;
    const int kv = blockIdx.y;
    const uint32_t t = row / (uint32_t)a.p.Hkv, h = row - t * a.p.Hkv;
    const int64_t from = slot_offset(a.p, a.lps, a.slots[t], h);
    u32x4 w = {0, 0, 0, 0};
    if (from >= 0) {
        if constexpr (!Q8) {
            w = *(const u32x4 *)((const uint16_t *)(kv ? a.p.v : a.p.k) + from + 8 * c);
        } else {
            const u32x2 q = *(const u32x2 *)((const uint8_t *)(kv ? a.p.v : a.p.k) + from + 8 * c);
            const int64_t g = (from + 8 * c) >> 6;
            const float s = f16bits_to_f32<BF>(((const uint16_t *)(kv ? a.p.v_scales : a.p.k_scales))[g]);
            const float b = f16bits_to_f32<BF>(((const uint16_t *)(kv ? a.p.v_biases : a.p.k_biases))[g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t two = q[i >> 1] >> (16 * (i & 1));
                w[i] = pack2<BF>(fmaf((float)(two & 0xFFu), s, b), fmaf((float)((two >> 8) & 0xFFu), s, b));
            }
        }
    }
    *(u32x4 *)(a.dst[kv] + (int64_t)row * D + 8 * c) = w;
}

template <int D, bool BF, bool Q8>
void launch_copy(const CopyArgs &a, bool write, hipStream_t s) {
    const dim3 grid((unsigned)(((uint64_t)a.rows * (D / 8) + 255) / 256), 2);
    if (write) hipLaunchKernelGGL((kq_paged_write_kernel<D, BF, Q8>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kq_paged_read_kernel<D, BF, Q8>), grid, dim3(256), 0, s, a);
}

template <int D>
void launch_copy_d(const CopyArgs &a, bool write, hipStream_t s) {
    const bool bf = a.p.dtype == KQ_DTYPE_BF16;
    if (a.p.k_scales) {
        if constexpr (D % 64 == 0) bf ? launch_copy<D, true, true>(a, write, s) : launch_copy<D, false, true>(a, write, s);
    } else {
        // a 16-bit row moves as bits whatever its type
        launch_copy<D, false, false>(a, write, s);
    }
}

int copy_rows(const CopyArgs &a, bool write, kq_stream_t stream) {
    // 32-bit item numbers
    if ((int64_t)a.T * a.p.Hkv * (a.p.D / 8) >= (int64_t)1 << 31) return KQ_ERR_BAD_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    switch (a.p.D) {
    case 64: launch_copy_d<64>(a, write, s); break;
    case 96: launch_copy_d<96>(a, write, s); break;
    case 128: launch_copy_d<128>(a, write, s); break;
    case 256: launch_copy_d<256>(a, write, s); break;
    default: launch_copy_d<512>(a, write, s); break;
    }
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

}  // namespace

extern "C" {

int kq_paged_plan(const int32_t *seq_lens, const int32_t *keep_lens, const int32_t *new_lens, int32_t B,
                  int32_t *block_table, int64_t table_stride, int32_t table_width, int32_t *free_pages,
                  int32_t n_stack, const int32_t *free_count, int32_t page_size, int32_t max_tokens, int32_t *cu_q,
                  int32_t *kv_lens, int32_t *slots, int32_t *positions, int32_t *free_count_out, int32_t *refused,
                  kq_stream_t stream) {
    if (!seq_lens || !new_lens || !block_table || !free_pages || !free_count || !cu_q || !kv_lens ||
        !free_count_out || !refused || (max_tokens > 0 && (!slots || !positions)))
        return KQ_ERR_NULL_POINTER;
    if (B < 1 || B > KQ_PAGED_MAX_ROWS || table_width < 1 || table_stride < table_width || n_stack < 0 ||
        max_tokens < 0)
        return KQ_ERR_BAD_SHAPE;
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return KQ_ERR_BAD_SHAPE;
    if ((int64_t)table_width * page_size >= (int64_t)1 << 31) return KQ_ERR_BAD_SHAPE;
    // 31-bit sums of pages, and numbers of tokens and pages a grid's step past the last
    if ((int64_t)B * table_width >= 1 << 30 || n_stack >= 1 << 30 || max_tokens > 1 << 30) return KQ_ERR_BAD_SHAPE;
    const PlanArgs a{seq_lens,       keep_lens, new_lens,     free_count,  block_table, free_pages,
                     cu_q,           kv_lens,   slots,        positions,   free_count_out, refused,
                     table_stride,   B,         table_width,  n_stack,     __builtin_ctz(page_size), max_tokens};
    const int grid = max_tokens <= kPlanThreads ? 1 : min((max_tokens + kPlanThreads - 1) / kPlanThreads, 64);
    hipLaunchKernelGGL(kq_paged_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

int kq_paged_write(const kq_paged_pool *pool, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                   const void *v, int64_t v_token_stride, int64_t v_head_stride, const int32_t *slots, int32_t T,
                   kq_stream_t stream) {
    if (const int rc = kq_pool_check(pool)) return rc;
    if (T == 0) return KQ_OK;
    if (!k || !v || !slots) return KQ_ERR_NULL_POINTER;
    if (T < 0) return KQ_ERR_BAD_SHAPE;
    if (!kq_pool_places_apart(*pool)) return KQ_ERR_BAD_ARGUMENT;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
        return KQ_ERR_BAD_ALIGN;
    const CopyArgs a{*pool,
                     {(const uint16_t *)k, (const uint16_t *)v},
                     {nullptr, nullptr},
                     {k_token_stride, v_token_stride},
                     {k_head_stride, v_head_stride},
                     slots,
                     T,
                     __builtin_ctz(pool->page_size),
                     (uint32_t)T * (uint32_t)pool->Hkv};
    return copy_rows(a, true, stream);
}

int kq_paged_read(const kq_paged_pool *pool, const int32_t *slots, int32_t T, void *k, void *v, kq_stream_t stream) {
    if (const int rc = kq_pool_check(pool)) return rc;
    if (T == 0) return KQ_OK;
    if (!k || !v || !slots) return KQ_ERR_NULL_POINTER;
    if (T < 0) return KQ_ERR_BAD_SHAPE;
    if (((uintptr_t)k | (uintptr_t)v) & 15) return KQ_ERR_BAD_ALIGN;
    const CopyArgs a{*pool,
                     {nullptr, nullptr},
                     {(uint16_t *)k, (uint16_t *)v},
                     {0, 0},
                     {0, 0},
                     slots,
                     T,
                     __builtin_ctz(pool->page_size),
                     (uint32_t)T * (uint32_t)pool->Hkv};
    return copy_rows(a, false, stream);
}

}  // extern "C"
