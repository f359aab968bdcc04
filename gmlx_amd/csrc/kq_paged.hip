// Attention of each row's new tokens over a paged KV cache (kq_sdpa_paged).
//
// A row's new tokens and the G = Hq / Hkv query heads that share a kv head are
// flattened to n * G query columns (column c: token c / G, head c % G).  Both
// products run on v_mfma_f32_16x16x32 with the query columns in the MFMA's
// columns:
//   S^T[tok, col] = K[tok, d] . q^T[d, col],  O^T[d, col] += V^T[d, tok] . P^T[tok, col]
// so that a lane's scores are the P.V operand it needs (lane 16 g + r holds
// column r at tokens 4g .. 4g+3 of each 16), and the softmax statistics of a
// column live in the four lanes that hold it.  One pass over the keys: a
// column's running maximum m, sum l of 2^(s - m) and sums O of 2^(s - m) v, all
// fp32; where a row is split, a merge adds the splits' (m, l, O) in split order.
//
// Rounded to 16 bits are the probabilities (an MFMA operand: half a step each,
// relative, averaged over the keys) and the output, nothing else; 8-bit pools
// multiply integers, or hi + lo planes of 21 bits (fp16) or 16 (bf16; the lost
// part is 2^-8 of half a step of the output).  Probabilities in hi + lo
// too would double P.V's products and take the error (2-norm, bf16) from 0.0023 to
// the 0.0017 of the output's own rounding.  In 8-bit fp16 decode rows a probability
// is rounded after its key's scale is on it: subnormal, so with fewer bits, where
// scales are below 1e-5 or so (values of 3e-4 behind a first key of e^10 times the
// others' weight: 7.6e-4 instead of the output rounding's 2.2e-4; of 1e-2: 2.1e-4).
//
// Few query columns (decode, verify): bound by HBM, one wave a unit streams its
// keys through registers; 16 rows of 1 k to 131 k keys, head dim 128, 2.01 GB
// in 371 us, 5.4 TB/s.  Chunks: bound by the MFMA, exp and LDS pipes together,
// tiles in LDS shared by the workgroup's columns; 2048 tokens behind 6000, head
// dim 128, 236 GFLOP in 247 to 277 us over cards and runs, 850 to 950 TFLOP/s (1.19
// PFLOP/s for a plain 8192^3 product on the card of the 247): MFMA pipes busy 45 % of
// the cycles, LDS 35 %, a third of that in bank conflicts.
#include "kq_once.h"
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
    int32_t group_cols, group_slots;
    int32_t few_limit;   // (few_columns)
    int32_t few_cols;    // a wave's 16, or group_cols where the chunks' kernel takes all rows
    float scale_log2;
    float *part, *ml;  // split partials: [slot][D] sums, [slot][2] (maximum, sum)
    SplitRule rule;    // rows of few columns
    // slots a token and query head, or 0: a row's slots follow those of the rows
    // before it (a chunk's tokens have fewer splits than a decode row's)
    int32_t slot_stride;
    int32_t slots;       // of the workspace
    int32_t few_blocks;  // the most 16-column blocks of a row of few columns
    int32_t direct;    // the wave kernel's grid is (split, kv head, row), the merge's (token and head, row)
    int32_t window, sinks;  // (Window)
};

// Least keys of a chunk's split, where the GPU has room for more workgroups: 512
// against 256 / 1024 (us): one chunk of 333 tokens over 4200 keys 50 / 50 / 54, 16
// over 4000 24 / 19 / 40, four of 100 over 1000 34 / 43 / 34, 8 rows of 8 over 2 k
// to 6 k 43 / 51 / 49, two chunks beside 14 decode rows 147 / 170 / 145.
constexpr int kSplitTokens = 512;
// Through a window, which has few splits of 512 (us with the merge, 512 against 256):
// rows of so few units that half the GPU is idle split at 256.  500 tokens through 777
// keys at head dim 256 49 / 43, 100 through 1000 at 128 33 / 29, 64 through 4000 35 / 31,
// 300 through 1000 in 8 bits at 256 67 / 52; but 1000 tokens through 500, 256 units, 33
// / 46.
constexpr int kLeastUnits = 128;
// Most waves, and merged tokens and heads, of grids in which each finds its place
// without a sum over the rows: three rows of 400 to 1700 keys 10.8 us (16.5 with
// the sum), 8 rows of 4 tokens 43.9 (45), four of 4000 at head dim 512 30 (38);
// beyond, waves without work cost more than the sums (16 rows of up to 131 k keys
// 398 against 395, 8-bit 241 against 237.5, at the limit).
constexpr int kDirect = 1 << 15;
constexpr int kMergeGroups = 1024;  // workgroups of a merge that is no such grid

// Rows of at most so many columns split as decode rows do and run in waves of 16
// columns.  Two waves read a row's keys twice, and still beat a chunk's
// workgroup with one of its waves at work where a tile costs conversions (8 bits:
// blocks of 5 tokens in 8 rows 45 us against 72) or the GPU is idle anyway (16
// bits: one row of 8 tokens and 4000 keys 14 against 24), but not where memory
// bounds them (16 bits, 8 rows: 55 against 42).
constexpr int few_limit(bool q8) { return q8 ? 32 : 16; }
__host__ __device__ __forceinline__ bool few_columns(int n, int G, int limit) { return (int64_t)n * G <= limit; }

// Whether such rows run a wave each (at head dim 512 a wave's tile, sums and query
// spill: the chunks' kernel takes all rows there).
constexpr bool has_waves(int D) { return D <= 256; }

// A chunk's workgroup: its waves (eight share an 8-bit tile's conversion: 333
// tokens over 4200 keys at head dim 256 142 us on four, 82 on eight (77 since
// fp16 halves are cut); at 128 85 and 73), query columns (32 a wave, 16 where 32
// would take over 256 registers a lane for the sums and the queries: at head dim
// 256 2048 tokens over 8048 keys 278 us, with 32 400), and how many such workgroups
// the GPU holds at once, which splitting a chunk aims at (512; half of it: 333 over
// 4200 50 -> 65).
constexpr int chunk_waves(int D, bool q8) { return q8 && (D == 128 || D == 256) ? 8 : 4; }
constexpr int group_columns(int D, bool q8) { return chunk_waves(D, q8) * (D > 128 ? 16 : 32); }
constexpr int group_slots(int D, bool q8) { return D > 256 || chunk_waves(D, q8) > 4 ? 256 : 512; }

// Blocks of `cols` query columns of a row.
__host__ __device__ __forceinline__ int row_blocks(int n, int G, int cols) {
    return (int)(((int64_t)n * G + cols - 1) / cols);
}

// Splits of a row of n tokens and kv keys: from the row and the head counts
// alone, so that a row of a batch has the bits of the row alone.
__host__ __device__ __forceinline__ int paged_splits(const SplitRule &rule, int n, int kv, int G, int Hkv, int few_limit,
                                                     int group_cols, int group_slots, int least_units) {
    if (few_columns(n, G, few_limit)) return row_splits(rule, kv);
    const int units = row_blocks(n, G, group_cols) * Hkv;
    return max(1, min(group_slots / units, kv / (units <= least_units ? kSplitTokens / 2 : kSplitTokens)));
}

struct Row {
    int q0;      // first query row
    int n;       // tokens computed
    int kv;      // keys attended: the row's, cut by max_kv and the table's width
    int span;    // keys that its splits divide: all, or the most that a block sees through its window
    int before;  // cached tokens before the new ones, uncut (below 0: more new ones than cached)
    int blocks, splits;
};

// A window: the token that sees keys 0 .. p alone sees the last `window` of them and
// the row's first `sinks`.  The keys that some column of a block sees are then its
// first `head` pieces of 16 (the sinks') and those from the first column's window
// on; the block numbers these keys on, as if the `skip` pieces between were not
// there, and everything that goes by key numbers (splits, tiles, ends) goes by
// these; only a table's entry and a key's place in its page go by the key itself.
// So what is read and multiplied is the window, whatever lies behind it.
struct Window {
    int head, skip;  // pieces of 16 keys

    // of a block whose first column sees `first` keys
    __device__ __forceinline__ Window(const PagedArgs &a, int first) {
        head = (a.sinks + 15) >> 4;
        skip = max((max(first - a.window, 0) >> 4) - head, 0);
    }
    // piece of the row that the block's piece c is
    __device__ __forceinline__ int piece(int c) const { return c < head ? c : c + skip; }
    // how many of the block's keys are among the row's first x
    __device__ __forceinline__ int keys(int x) const { return x <= 16 * head ? x : max(16 * head, x - 16 * skip); }
    // the first key of the block in the window of a token that sees `seen` keys
    __device__ __forceinline__ int low(const PagedArgs &a, int seen) const { return keys(max(seen - a.window, 0)); }
};

// The most keys that a block of `cols` columns of up to n tokens sees through a
// window (its tokens' windows together, with what completes the pieces at the ends).
__host__ __device__ __forceinline__ int window_span(int kv, int window, int sinks, int n, int G, int cols) {
    const int tokens = (cols + G - 2) / G + 1;
    const int64_t span = (int64_t)((sinks + 15) & ~15) + window + (n < tokens ? n : tokens) + 14;
    return (int)(span < kv ? span : kv);
}

template <bool WIN>
__device__ __forceinline__ Row row_at(const PagedArgs &a, int b) {
    Row r;
    r.q0 = min(max(a.cu_q[b], 0), a.T);
    const int n = min(max(a.cu_q[b + 1], r.q0), a.T) - r.q0, kv = max(a.kv_lens[b], 0);
    r.n = min(n, a.max_q);
    r.kv = (int)min((int64_t)min(kv, a.max_kv), (int64_t)a.width << a.lps);
    // what a token sees goes by the row as it is, of which a cut leaves keys out
    r.before = kv - n;
    const int cols = few_columns(r.n, a.G, a.few_limit) ? a.few_cols : a.group_cols;
    r.blocks = row_blocks(r.n, a.G, cols);
    r.span = r.kv;
    if constexpr (WIN) {
        // (keys that only tokens past max_q see are nobody's)
        r.kv = min(r.kv, max(r.before + r.n, 0));
        r.span = window_span(r.kv, a.window, a.sinks, r.n, a.G, cols);
    }
    r.splits = paged_splits(a.rule, r.n, r.span, a.G, a.Hkv, a.few_limit, a.group_cols, a.group_slots, WIN ? kLeastUnits : 0);
    return r;
}

// Units of the wave kernel, of the chunk kernel, and of the merge (merge_items
// tokens and query heads of a row that has splits).
__device__ __forceinline__ int wave_units(const PagedArgs &a, const Row &r) {
    return few_columns(r.n, a.G, a.few_limit) ? r.blocks * r.splits * a.Hkv : 0;
}
template <int D>
__device__ __forceinline__ int chunk_units(const PagedArgs &a, const Row &r) {
    return has_waves(D) && few_columns(r.n, a.G, a.few_limit) ? 0 : r.blocks * r.splits * a.Hkv;
}
// A workgroup's share of a merge: a quarter of one item where all its threads add up
// its splits (one row of 131072 keys 105 us, a whole item a workgroup 113),
// one a wave where a wave takes several rounds of loads for them, four a wave,
// each loaded ahead of the one before, where it takes one (500 tokens in 4 splits
// beside decode rows 68 us; with one a wave there too 73).
constexpr int kSlices = 4;
__device__ __forceinline__ int merge_items(int splits) { return splits > 8 ? 4 : 16; }
__device__ __forceinline__ int merge_units(const PagedArgs &a, const Row &r) {
    if (r.splits > 64) return r.n * a.Hq * kSlices;
    const int items = merge_items(r.splits);
    return r.splits > 1 ? (r.n * a.Hq + items - 1) / items : 0;
}

// (the host refuses calls whose unit or slot numbers pass 31 bits)
__device__ __forceinline__ int row_slots(const PagedArgs &a, const Row &r) {
    return r.splits > 1 ? r.n * a.Hq * r.splits : 0;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return v;
}

// Largest over the wave's lanes, in scalar registers.
__device__ __forceinline__ float wave_max(float v) {
    const auto step = [&](auto ctrl, auto rows) {
        const int low = __builtin_bit_cast(int, -INFINITY);
        v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(low, __builtin_bit_cast(int, v), ctrl.value,
                                                                          rows.value, 0xf, false)));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr:1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15, 31
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Partial slot of split 0 of token i (of the row), query head hq.
__device__ __forceinline__ int64_t slot_of(const PagedArgs &a, const Row &r, int slot0, int i, int hq) {
    if (a.slot_stride) return ((int64_t)(r.q0 + i) * a.Hq + hq) * a.slot_stride;
    return slot0 + (i * a.Hq + hq) * r.splits;
}

// Whether a row's partials lie in the workspace: its size counts every query row
// once, and a cu_q that runs backwards may count some twice.  Such rows are left
// out, by all kernels alike (the row is the same in a whole workgroup).
__device__ __forceinline__ bool has_slots(const PagedArgs &a, const Row &r, int slot0) {
    return a.slot_stride || r.splits <= 1 || (slot0 >= 0 && slot0 <= a.slots - row_slots(a, r));
}

// Row x of lane src, in scalar registers.
__device__ __forceinline__ Row lane_row(const Row &x, int src) {
    Row r;
    r.q0 = __builtin_amdgcn_readlane(x.q0, src);
    r.n = __builtin_amdgcn_readlane(x.n, src);
    r.kv = __builtin_amdgcn_readlane(x.kv, src);
    r.span = __builtin_amdgcn_readlane(x.span, src);
    r.before = __builtin_amdgcn_readlane(x.before, src);
    r.blocks = __builtin_amdgcn_readlane(x.blocks, src);
    r.splits = __builtin_amdgcn_readlane(x.splits, src);
    return r;
}

// The row b that unit u belongs to, with u made its number within the row, and
// the row's first partial slot; false past the last unit.  units(row) is summed
// over the rows, 64 at a time, by every wave that asks.
template <bool WIN, class Units>
__device__ __forceinline__ bool find_unit(const PagedArgs &a, Units &&units, int &u, int &b, Row &row, int &slot0) {
    const int lane = kq_lane();
    int slots = 0;
    for (int c0 = 0; c0 < a.B; c0 += 64) {
        int mu = 0, ms = 0;
        Row x{};
        if (c0 + lane < a.B) {
            x = row_at<WIN>(a, c0 + lane);
            mu = units(x);
            ms = row_slots(a, x);
        }
        const int iu = wave_scan(mu), is = wave_scan(ms);
        const int total = __builtin_amdgcn_readlane(iu, 63);
        if (u < total) {
            const int src = __builtin_ctzll(__ballot(u < iu));
            b = c0 + src;
            u -= __builtin_amdgcn_readlane(iu - mu, src);
            slot0 = slots + __builtin_amdgcn_readlane(is - ms, src);
            row = lane_row(x, src);
            return true;
        }
        u -= total;
        slots += __builtin_amdgcn_readlane(is, 63);
    }
    return false;
}

// 64 entries of a block table row in a register; at(p) takes rising p.
struct PageIds {
    int first, ids;

    // Whether the entries first .. last all are pages of the pool.
    __device__ __forceinline__ static bool all_pages(const PagedArgs &a, const int32_t *tab, int first, int last) {
        bool bad = false;
        for (int i = first; i <= last; i += 64) bad |= (uint32_t)tab[min(i + kq_lane(), last)] >= (uint32_t)a.n_pages;
        return __builtin_amdgcn_ballot_w64(bad) == 0;
    }

    // Whether those of pieces c0 .. c1 of 16 keys (1 << sh a page) through a window
    // are; loads the first 64.
    __device__ __forceinline__ bool start(const PagedArgs &a, const int32_t *tab, const Window &win, int c0, int c1, int sh) {
        load(tab, win.piece(c0) >> sh, win.piece(c1) >> sh);
        return (c0 >= win.head || all_pages(a, tab, c0 >> sh, min(c1, win.head - 1) >> sh)) &&
               (c1 < win.head || all_pages(a, tab, win.piece(max(c0, win.head)) >> sh, win.piece(c1) >> sh));
    }

    // Whether entries p .. last all are pages of the pool; loads the first 64.
    __device__ __forceinline__ bool start(const PagedArgs &a, const int32_t *tab, int p, int last) {
        load(tab, p, last);
        bool bad = (uint32_t)ids >= (uint32_t)a.n_pages;
        // (every lane in every round: where lanes left such a loop one by one, the
        // compiler has put register copies before the restore of EXEC behind it)
        for (int i = p + 64; i <= last; i += 64)
            bad |= (uint32_t)tab[min(i + kq_lane(), last)] >= (uint32_t)a.n_pages;
        return __builtin_amdgcn_ballot_w64(bad) == 0;
    }

    __device__ __forceinline__ void load(const int32_t *tab, int p, int last) {
        first = p;
        ids = tab[min(p + kq_lane(), last)];
        // waited for here: after a branch that may load them, the compiler
        // would wait for every load in flight (a tile) before each use
        __builtin_amdgcn_s_waitcnt(KQ_VMCNT(0));
    }
    __device__ __forceinline__ int at(const int32_t *tab, int p, int last) {
        if ((uint32_t)(p - first) >= 64u) load(tab, p, last);
        return __builtin_amdgcn_readlane(ids, p - first);
    }
};

// 16-bit values whose exponent is all ones (infinities and NaN) as 0 in a
// masked tile: there the product of a hidden key's value with its probability
// 0 would be NaN.  `odd` collects whether there were any; the columns that see
// one get it from add_odd.
template <bool BF>
__device__ __forceinline__ uint32_t finite2(uint32_t x, uint32_t &odd) {
    constexpr uint32_t kExp = BF ? 0x7F807F80u : 0x7C007C00u, kStep = BF ? 0x00800080u : 0x04000400u;
    const uint32_t top = ((x & kExp) + kStep) & 0x80008000u;  // exponent + 1 carries into the sign's place
    odd |= top;
    return x & ~(top | (top - (top >> 15)));
}

// What an infinite or NaN value that a column sees does to its sum, else 0.
template <bool BF>
__device__ __forceinline__ float odd_part(uint32_t x) {
    const float v = f16bits_to_f32<BF>(x);
    return v - v == 0.f ? 0.f : v;
}

// Exponent shift of the probabilities: they and their sum are 2^kShift times
// the softmax's, which keeps fp16 ones of far smaller keys out of the
// subnormals; the quotient is the same.  An 8-bit cache multiplies a
// probability by its key's scale (up to 514) before it is rounded.
template <bool BF, bool Q8>
constexpr float shift() { return BF ? 0.f : Q8 ? 6.f : 10.f; }

template <int D>
struct Geo {
    static constexpr int TT = 32;       // tokens a tile
    static constexpr int CH = TT / 16;  // 16-token chunks
    static constexpr int VT = TT / 4;   // V rows a lane
    static constexpr int NC = D / 32;   // 32-wide pieces of the head dim
};

// Where a tile's chunks start in the pool (elements or bytes; uniform), and
// which of them lie in a page of the pool.
template <int D>
struct TileAt {
    int64_t off[Geo<D>::CH];
    uint32_t ok;  // bit ch
};

// One tile in registers, 16-bit pool.
template <int D, bool BF>
struct Tile16 {
    static constexpr int CH = Geo<D>::CH, VT = Geo<D>::VT, NC = Geo<D>::NC, NG = (D + 127) / 128;
    u32x4 k[CH][NC];  // token 16 ch + r, d = 32 c + 8 g .. +7
    u32x4 v[NG][VT];  // token 4g + i | 16 + 4g + i - 4, d = 128 dg + 8 r .. +7

    __device__ __forceinline__ void load(const PagedArgs &a, const TileAt<D> &at) {
        const int lane = kq_lane(), r = lane & 15, g = lane >> 4;
        // uniform bases and 32-bit byte offsets of the lanes
        const uint32_t ko = 2u * (uint32_t)(r * a.tok_stride + 8 * g), vo = 2u * (uint32_t)(4 * g * a.tok_stride);
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
            const uint8_t *kp = (const uint8_t *)a.k + 2 * at.off[ch];
#pragma unroll
            for (int c = 0; c < NC; ++c) k[ch][c] = *(const u32x4 *)(kp + 64 * c + ko);
        }
#pragma unroll
        for (int i = 0; i < VT; ++i) {
            const uint8_t *vp = (const uint8_t *)a.v + 2 * (at.off[i >> 2] + (i & 3) * a.tok_stride);
#pragma unroll
            for (int dg = 0; dg < NG; ++dg)
                v[dg][i] = *(const u32x4 *)(vp + 256 * dg + (vo + 2u * (uint32_t)min(8 * r, D - 8 - 128 * dg)));
        }
    }
};

// 8 bytes as 16-bit floats of their integer values less Z (0 or 128), exactly.
template <bool BF, int Z>
__device__ __forceinline__ u32x4 bytes8(u32x2 q) {
    static_assert(Z == 0 || Z == 128, "as they are, or signed");
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
            float x, y;
            if constexpr (Z == 0) {
                x = (float)((w >> (8 * j)) & 0xFFu);
                y = (float)((w >> (8 * j + 8)) & 0xFFu);
            } else {  // (signed bytes convert in one step)
                x = (float)(int8_t)(w >> (8 * j));
                y = (float)(int8_t)(w >> (8 * j + 8));
            }
            return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
        };
        if constexpr (Z != 0) q = u32x2{q.x ^ 0x80808080u, q.y ^ 0x80808080u};
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
                const u32x4 w = *(const u32x4 *)(kp + 64 * i + (uint32_t)(r * D + 16 * g));
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
                v[grp][i] = *(const uint32_t *)((const uint8_t *)a.v + at.off[i >> 2] + ((i & 3) * D + 64 * grp) +
                                                (uint32_t)(4 * g * D + 4 * r));
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
    __device__ __forceinline__ void tile(const Tile &t, float scale_log2, uint32_t vis, uint32_t &odd) {
        float s[8];
        scores(t, scale_log2, s);
        constexpr int N = 8;
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
        for (int j = 0; j < N; ++j) p[j] = __builtin_amdgcn_exp2f(s[j] - (m_use - shift<BF, Q8>()));
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
            pv16<MASK>(t, p, odd);
        } else {
#pragma unroll
            for (int grp = 0; grp < SG; ++grp) {
                float ps[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
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
                for (int i = 0; i < 8; ++i) w[i] = t.v[grp][i];
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
    __device__ __forceinline__ void pv16(const Tile &t, const float (&p)[8], uint32_t &odd) {
        const half8_t pf = __builtin_bit_cast(half8_t, u32x4{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3]),
                                                             pack2<BF>(p[4], p[5]), pack2<BF>(p[6], p[7])});
#pragma unroll
        for (int dg = 0; dg < Tile::NG; ++dg) {
            u32x4 vr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                vr[i] = t.v[dg][i];
                if constexpr (MASK) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) vr[i][w] = finite2<BF>(vr[i][w], odd);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                u32x4 f;
                f.x = __builtin_amdgcn_perm(vr[1][j >> 1], vr[0][j >> 1], sel);
                f.y = __builtin_amdgcn_perm(vr[3][j >> 1], vr[2][j >> 1], sel);
                f.z = __builtin_amdgcn_perm(vr[5][j >> 1], vr[4][j >> 1], sel);
                f.w = __builtin_amdgcn_perm(vr[7][j >> 1], vr[6][j >> 1], sel);
                o[dg * 8 + j] = mfma<BF>(__builtin_bit_cast(half8_t, f), pf, o[dg * 8 + j]);
            }
        }
    }

    // Adds the infinite and NaN values of one key (its row of V) to the columns
    // that see it.
    __device__ __forceinline__ void add_odd(const uint16_t *v, bool sees) {
        const int g = kq_lane() >> 4;
#pragma unroll
        for (int j = 0; j < NO; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (results past D are not stored)
                const float x = odd_part<BF>(v[min(128 * (j >> 3) + 8 * (4 * g + e) + (j & 7), D - 1)]);
                o[j][e] += sees ? x : 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);  // (few loads at a time: registers)
        }
    }
};

// Rows of few columns: one wave a unit = (row, split, kv head), the kv heads
// fastest.  The wave takes the units `first`, `first` + `step`, ..., or with
// DIRECT the one of its place in the grid.
template <int D, bool BF, bool Q8, bool DIRECT, bool WIN>
__device__ __forceinline__ void wave_work(const PagedArgs &a, int first, int step) {
    using Tile = std::conditional_t<Q8, Tile8<D, BF>, Tile16<D, BF>>;
    constexpr int TT = Geo<D>::TT, CH = Geo<D>::CH, NC = Geo<D>::NC;
    constexpr int NBUF = D >= 256 ? 1 : 2;
    const int lane = kq_lane(), r = lane & 15, g = lane >> 4;
    for (int unit = first;; unit += step) {
        // the 16-column blocks of a row (at most two) read the same keys: one after
        // the other in the scan's order, eight apart, on one XCD, in the grid's
        int b, h, s, blk, slot0 = 0;
        Row row;
        if constexpr (DIRECT) {
            if (unit >= step) return;  // (one unit a wave)
            s = a.few_blocks > 1 ? unit / 16 * 8 + unit % 8 : unit;
            blk = a.few_blocks > 1 ? unit / 8 % 2 : 0;
            h = blockIdx.y;
            b = blockIdx.z;
            // Rows with fewer splits than the grid has leave its last places idle: turned
            // by row and head, these fall on all XCDs alike (64 rows of 5 splits in a grid
            // of 8, the XCD's number in place of the split's: 39 us, unturned 49)
            const int most = a.few_blocks > 1 ? gridDim.x / 2 : gridDim.x;
            s += (h + b * a.Hkv) & 7;
            while (s >= most) s -= most;
            row = lane_row(row_at<WIN>(a, b), 0);
            if (!few_columns(row.n, a.G, a.few_limit) || blk >= row.blocks || s >= row.splits) return;
        } else {
            int u = unit;
            if (!find_unit<WIN>(a, [&](const Row &x) { return wave_units(a, x); }, u, b, row, slot0)) return;
            if (!has_slots(a, row, slot0)) continue;
            const int head = u / row.blocks;
            blk = u - head * row.blocks;
            s = head / a.Hkv;
            h = head - s * a.Hkv;
        }

        // this lane's column
        const int col = 16 * blk + r;
        const bool live = col < row.n * a.G;
        const int i = live ? col / a.G : row.n - 1, hq = h * a.G + (live ? col - i * a.G : 0);
        State<D, BF, Q8> st;
        st.init();
        // keys seen: the column's, the block's least and most
        const int first = row.before + 1;
        int seen = live ? max(first + i, 0) : 0x7fffffff;
        int least = max(first + 16 * blk / a.G, 0);
        int most = min(max(first + min((16 * blk + 15) / a.G, row.n - 1), 0), row.kv);
        // with a window, by the block's numbers: the column's first key behind the
        // sinks, and the block's last such (a dead column may see any)
        const Window win(a, WIN ? least : 0);
        int low = 0, low_all = 0;
        if constexpr (WIN) {
            low = live ? win.low(a, seen) : 0;
            low_all = __builtin_amdgcn_readfirstlane(win.low(a, max(first + min((16 * blk + 15) / a.G, row.n - 1), 0)));
            seen = live ? win.keys(min(seen, row.kv)) : seen;
            least = win.keys(min(least, row.kv));
            most = win.keys(most);
        }
        const auto in_window = [&](int t) { return !WIN || t < a.sinks || t >= low; };
        const int per = a.rule.tokens(row.span);
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
            const int c_last = (t_end - 1) >> 4, p_last = (WIN ? win.piece(c_last) : c_last) >> sh;
            PageIds ids;
            bool all_ok;
            if constexpr (WIN) all_ok = ids.start(a, tab, win, t_begin >> 4, c_last, sh);
            else all_ok = ids.start(a, tab, (t_begin >> 4) >> sh, p_last);
            const int64_t h_off = (int64_t)h * a.head_stride;
            auto at_tile = [&](int t0) {
                TileAt<D> x;
                x.ok = 0;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) {
                    // (chunks past the end repeat the last: their keys are hidden)
                    const int cb = min((t0 >> 4) + ch, c_last), c = WIN ? win.piece(cb) : cb, p = c >> sh;
                    const int id = ids.at(tab, p, p_last);
                    const bool in = (uint32_t)id < (uint32_t)a.n_pages;
                    x.ok |= in ? 1u << ch : 0u;
                    x.off[ch] = uniform64((int64_t)(in ? id : 0) * a.page_stride + h_off +
                                          (int64_t)((c - (p << sh)) * 16) * a.tok_stride);
                }
                return x;
            };
            // Tiles that every column sees whole run through the ring; the
            // others (the last keys; all, where the table names no page) one
            // by one before them, so that their code is there once.
            int whole = min(least, t_end);
            whole = whole <= t_begin || !all_ok ? t_begin : whole - (whole - t_begin) % TT;
            // With a window only those below `sunk` (sinks) and from `from` on are whole.
            int sunk = t_begin, from = t_begin;
            if constexpr (WIN) {
                const int head = min(a.sinks, whole), all = min(low_all, whole);
                sunk += max(head - t_begin, 0) / TT * TT;
                from = max(sunk, t_begin + (max(all - t_begin, 0) + TT - 1) / TT * TT);
            }
            const int n_sunk = (sunk - t_begin) / TT;
            // (tile k of the whole ones)
            const auto whole_at = [&](int k) { return !WIN || k < n_sunk ? t_begin + TT * k : from + TT * (k - n_sunk); };
            const int n_whole = WIN ? n_sunk + (whole - from) / TT : (whole - t_begin) / TT;
            Tile ring[NBUF];
#pragma unroll 1
            for (int t = WIN && sunk < from ? sunk : whole; t < t_end; t += TT) {
                if constexpr (WIN) {
                    if (t == from && t < whole) t = whole;
                    if (t >= t_end) break;
                }
                const TileAt<D> at = at_tile(t);
                ring[0].load(a, at);
                const int lim = min(seen, t_end);
                uint32_t vis = 0, odd = 0;
#pragma unroll
                for (int x = 0; x < 4 * CH; ++x)
                    if (((at.ok >> (x >> 2)) & 1) && t + 16 * (x >> 2) + 4 * g + (x & 3) < lim &&
                        in_window(t + 16 * (x >> 2) + 4 * g + (x & 3)))
                        vis |= 1u << x;
                st.template tile<true>(ring[0], a.scale_log2, vis, odd);
                if constexpr (!Q8) {
                    if (__builtin_amdgcn_ballot_w64(odd != 0)) {
#pragma unroll 1
                        for (int k = 0; k < TT; ++k)
                            st.add_odd((const uint16_t *)a.v + (k < 16 ? at.off[0] : at.off[1]) + (k & 15) * a.tok_stride,
                                       ((at.ok >> (k >> 4)) & 1) && t + k < lim && in_window(t + k));
                    }
                }
            }
            if (n_whole > 0) {
                uint32_t odd;
#pragma unroll
                for (int j = 0; j < NBUF - 1; ++j) ring[j].load(a, at_tile(whole_at(j)));
                for (int k = 0; k < n_whole; k += NBUF) {
#pragma unroll
                    for (int j = 0; j < NBUF; ++j) {
                        ring[(j + NBUF - 1) % NBUF].load(a, at_tile(whole_at(k + j + NBUF - 1)));
                        __builtin_amdgcn_sched_barrier(0);
                        if (k + j < n_whole) st.template tile<false>(ring[j], a.scale_log2, 0, odd);
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
        const int64_t slot = slot_of(a, row, slot0, i, hq) + s;
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

template <int D, bool BF, bool Q8, bool DIRECT, bool WIN>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void kq_paged_wave_kernel(
    PagedArgs a) {
    wave_work<D, BF, Q8, DIRECT, WIN>(a, blockIdx.x, gridDim.x);
}

// ---- prompt chunks --------------------------------------------------------
// Rows of more query columns: a workgroup takes 128 (64 for 16-bit pools past
// head dim 128, 256 for 8-bit ones at 128), 32 or 16 a wave, and streams the keys
// in tiles of BN tokens through two LDS stages, copied by direct-to-LDS loads one
// tile ahead; one barrier a tile.
// v_mfma_f32_32x32x16: lane 32 h + c holds column c at tokens 8 (i / 4) + 4 h +
// i % 4 (i < 16) of each 32, which are the P.V operand's eight tokens a lane of
// two 16-token products; V's operand, eight tokens of one head dim a lane, is
// read from the row-major tile by transposing LDS reads (ds_read_b64_tr_b16:
// each group of 16 lanes reads 4 tokens x 16 values and gets a column a lane).
//
// An 8-bit pool's tile is written to LDS as 16-bit values by the waves that
// would copy it: value = hi + lo, each in the queries' type, hi the value
// s q + b in 16 bits and lo the rest, both multiplied (twice the MFMAs), so that
// no rounding of a dequantised value to 16 bits enters the result; dequantised
// to hi alone, outputs were about twice as far from exact as the 16-bit pool's.
// A value past the largest fp16 (255 steps from the least to 65504 end at 65535)
// has that as hi and the rest as lo.
template <int D, bool Q8>
struct Chunk {
    static constexpr int NW = chunk_waves(D, Q8);                      // waves
    static constexpr int NP = Q8 ? 2 : 1;                              // planes: the values, or hi and lo
    static constexpr int BN = D * NP <= 128 ? 64 : 32;                 // tokens a tile
    static constexpr int NT = BN / 32;                                 // 32-token blocks
    static constexpr int RC = D / 8;                                   // 16-byte pieces of a token's row
    static constexpr int kRow = 2 * D;                                 // bytes
    static constexpr int kPlane = BN * kRow;                           // K or V of a tile
    static constexpr int kHalf = NP * kPlane;                          // V's place behind K's
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kStages = 2 * kStage <= (160 << 10) ? 2 : 1;  // (8-bit rows of 512: one)
    static constexpr int kLds = kStages * kStage;
    static constexpr int kCopies = 16 * RC / 64;                       // 1 KB loads of 16 tokens

    // Rows lie as they are but for the order of their pieces: piece c of row t
    // is at place c ^ f(t), so that the 16 rows an operand read touches at one
    // c lie in different banks.  K: single pieces; V: pairs (a transposing read
    // takes 32 bytes of a row).
    // So the piece's number enters the address by XOR in the swizzled bits (kSw)
    // and by addition above them, the same for every lane.
    static constexpr int kSw = D == 64 ? 7 : D == 96 ? 3 : 15;
    __device__ __forceinline__ static int kswz(int t) {
        return D == 64 ? (t >> 1) & 7 : D == 96 ? (t >> 2) & 3 : t & 15;
    }
    __device__ __forceinline__ static int vswz(int t) {
        return D == 64 ? ((t >> 1) & 3) << 1 : D == 96 ? ((t >> 2) & 1) << 1 : (t & 7) << 1;
    }
};

typedef float floatx16 __attribute__((ext_vector_type(16)));

template <bool BF>
__device__ __forceinline__ floatx16 mfma32(const half8_t &a, const half8_t &b, const floatx16 &c) {
    if constexpr (!BF) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    } else {
        typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
}

#define LDSP(T) __attribute__((address_space(3))) T *

__device__ __forceinline__ half8_t lds_half8(uint32_t at) {
    return __builtin_bit_cast(half8_t, *(const LDSP(u32x4))(uintptr_t)at);
}

// Four tokens of one head dim a lane from a row-major tile.
__device__ __forceinline__ u32x2 lds_tr(uint32_t at, uint32_t more) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDSP(s16x4))(uintptr_t)at + more / 8));
}

// 16 bytes a lane from base + off straight to LDS, lane l's at lds + 16 l (the
// base in m0, which the compiler sets).  Written out because the compiler
// orders every LDS read behind the builtin's copy and would wait for the next
// tile before the first operand of this one; the wait is the one at the tile's
// barrier.
__device__ __forceinline__ void copy16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds), "v"(off), "s"(base) : "memory");
}

__device__ __forceinline__ float other_half_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// mfma(i, operand) for i < N with the operands read AHEAD steps before their
// use, so that no MFMA waits for a read that was just issued (left alone, the
// scheduler saves registers and puts every read right before its MFMA).  Reads
// and MFMAs keep this order; vector and scalar ALU work may move across.  The
// wave goes before the SIMD's other one meanwhile, whose softmax then fills the
// gaps (a 2048-token chunk 257 -> 251 us).
template <int N, int AHEAD, class Read, class Use>
__device__ __forceinline__ void pipelined(Read &&read, Use &&use) {
    constexpr int A = AHEAD < N ? AHEAD : N;
    half8_t f[A + 1];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < A; ++i) f[i] = read(i);
    __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i + A < N) f[(i + A) % (A + 1)] = read(i + A);
        __builtin_amdgcn_sched_barrier(0x6);
        use(i, f[i % (A + 1)]);
        __builtin_amdgcn_sched_barrier(0x6);
    }
    __builtin_amdgcn_s_setprio(0);
}

// How far (log2) a tile's maximum may pass the one that the sums are held at
// before they are rescaled: the probabilities stay below 2^(shift + slack).
template <bool BF>
constexpr float slack() { return BF ? 8.f : 4.f; }

// Which keys of a tile a lane's column sees, by their distance from the lane's
// first key t: below lim, and through a window below sinks or from low on.
struct Shown {
    int end, sunk, from;
    __device__ __forceinline__ Shown(int t, int lim, int sinks, int low) : end(lim - t), sunk(sinks - t), from(low - t) {}
    template <bool WIN>
    __device__ __forceinline__ bool at(int d) const {
        return d < end && (!WIN || d < sunk || d >= from);
    }
};

template <int D, bool BF, bool Q8>
struct ChunkState {
    using C = Chunk<D, Q8>;
    static constexpr int COLS = 32, NQ = D / 16, ND = D / 32;
    static constexpr int NR = D / 8;  // runs of four results a lane
    half8_t qf[NQ];
    floatx16 o[ND];
    float m_run, l_part;

    __device__ __forceinline__ static int qd(int d) { return 16 * d + 8 * (kq_lane() >> 5); }
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) o[j][x] = 0.f;
        m_run = -INFINITY;
        l_part = 0.f;
    }
    __device__ __forceinline__ float sum() const { return l_part + __shfl_xor(l_part, 32); }
    // results d .. d + 3 of run k
    __device__ __forceinline__ static int run_d(int k) { return 8 * k + 4 * (kq_lane() >> 5); }
    __device__ __forceinline__ floatx4 run(int k) const {
        const int j = k >> 2, x = 4 * (k & 3);
        return floatx4{o[j][x], o[j][x + 1], o[j][x + 2], o[j][x + 3]};
    }
    __device__ __forceinline__ void add(int k, const floatx4 &y) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k >> 2][4 * (k & 3) + e] += y[e];
    }

    // masked: some key of the tile is hidden from a column (lim: the column's
    // first unseen key; with a window, it sees below `sinks` and from `low` on; okbits:
    // the 16-token pieces that lie in the pool).
    template <bool WIN>
    __device__ __forceinline__ void tile(uint32_t stage, float scale_log2, bool masked, int t0, int lim, int sinks, int low,
                                         uint32_t okbits) {
        const int lane = kq_lane(), c = lane & 31, h = lane >> 5;
        floatx16 s[C::NT];
        // rows t and t + 32 have the same order of pieces
        const uint32_t ka = stage + (uint32_t)(c * C::kRow) + 16u * (uint32_t)(C::kswz(c) ^ h);
#pragma unroll
        for (int b = 0; b < C::NT; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
        // operand x: head dims 16 d .. (d slowest), plane, 32-token block
        pipelined<NQ * C::NP * C::NT, 4>(
            [&](int x) {
                const int b = x % C::NT, pl = x / C::NT % C::NP, d = x / (C::NT * C::NP);
                const uint32_t kd = (ka ^ (uint32_t)(16 * ((2 * d) & C::kSw))) + (uint32_t)(16 * ((2 * d) & ~C::kSw));
                return lds_half8(kd + (uint32_t)(pl * C::kPlane + 32 * b * C::kRow));
            },
            [&](int x, const half8_t &f) { s[x % C::NT] = mfma32<BF>(f, qf[x / (C::NT * C::NP)], s[x % C::NT]); });
        if (masked) {
            const Shown shown(t0 + 4 * h, lim, sinks, low);
#pragma unroll
            for (int b = 0; b < C::NT; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[b][i] = shown.template at<WIN>(32 * b + 8 * (i >> 2) + (i & 3)) ? s[b][i] : -INFINITY;
            if (okbits != (1u << 2 * C::NT) - 1) {
#pragma unroll
                for (int b = 0; b < C::NT; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[b][i] = (okbits >> (2 * b + (i >> 3))) & 1 ? s[b][i] : -INFINITY;
            }
        }
        float tmax = s[0][0];
#pragma unroll
        for (int b = 0; b < C::NT; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) tmax = max3(tmax, s[b][i], s[b][i + 1]);
        tmax = other_half_max(tmax) * scale_log2;
        // (each column by its own scores: what the others see does not matter)
        const bool up = tmax > m_run + slack<BF>();
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float alpha = up ? __builtin_amdgcn_exp2f(m_run - tmax) : 1.f;
            m_run = up ? tmax : m_run;
            l_part *= alpha;
#pragma unroll
            for (int j = 0; j < ND; ++j) o[j] = o[j] * alpha;
        }
        // (no key yet: every power is 0, not exp(-inf + inf))
        const float m_use = (m_run == -INFINITY ? 0.f : m_run) - shift<BF, false>();
        half8_t pf[2 * C::NT];
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2 * C::NT; ++k) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(s[k >> 1][8 * (k & 1) + i], scale_log2, -m_use));
                sums[i & 3] += p[i];
            }
            pf[k] = __builtin_bit_cast(half8_t, u32x4{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3]),
                                                      pack2<BF>(p[4], p[5]), pack2<BF>(p[6], p[7])});
        }
        l_part += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        // lane 16 g + i: token 4 h + i / 4 (+ 8), values 32 j + 16 (g % 2) + 4 (i % 4) ..
        const uint32_t vt = stage + C::kHalf;
        const int tr = 4 * h + ((lane >> 2) & 3);
        const int piece = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        const uint32_t va = vt + (uint32_t)(tr * C::kRow) + 16u * (uint32_t)(C::vswz(tr) ^ piece) + 8u * (lane & 1);
        // (rows 8 apart have the same order of pieces but for head dims 64 and 96)
        const uint32_t vb = vt + (uint32_t)((tr + 8) * C::kRow) + 16u * (uint32_t)(C::vswz(tr + 8) ^ piece) + 8u * (lane & 1);
        // operand x: 16 tokens kk (slowest), plane, head dims 32 j ..
        pipelined<2 * C::NT * ND * C::NP, 4>(
            [&](int x) {
                const int j = x % ND, pl = x / ND % C::NP, kk = x / (ND * C::NP);
                const uint32_t flip = 16 * ((4 * j) & C::kSw);
                const uint32_t up = 16 * ((4 * j) & ~C::kSw) + 16 * kk * C::kRow + pl * C::kPlane;
                const u32x2 a = lds_tr(va ^ flip, up), b = lds_tr(vb ^ flip, up);
                return __builtin_bit_cast(half8_t, u32x4{a.x, a.y, b.x, b.y});
            },
            [&](int x, const half8_t &f) { o[x % ND] = mfma32<BF>(f, pf[x / (ND * C::NP)], o[x % ND]); });
        kq_mfma_drain();
    }
};

// The same for 16 columns a wave on v_mfma_f32_16x16x32 (head dims past 128):
// lane 16 g + c holds column c at tokens 4 g .. 4 g + 3 of each 16.
template <int D, bool BF, bool Q8>
struct ChunkState16 {
    using C = Chunk<D, Q8>;
    static_assert(C::BN == 32, "one product of 32 tokens a tile");
    static constexpr int COLS = 16, NQ = D / 32, NR = D / 16;
    half8_t qf[NQ];
    floatx4 o[NR];
    float m_run, l_part;

    __device__ __forceinline__ static int qd(int d) { return 32 * d + 8 * (kq_lane() >> 4); }
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int j = 0; j < NR; ++j) o[j] = floatx4{0, 0, 0, 0};
        m_run = -INFINITY;
        l_part = 0.f;
    }
    __device__ __forceinline__ float sum() const {
        const float l = l_part + __shfl_xor(l_part, 16);
        return l + __shfl_xor(l, 32);
    }
    __device__ __forceinline__ static int run_d(int k) { return 16 * k + 4 * (kq_lane() >> 4); }
    __device__ __forceinline__ floatx4 run(int k) const { return o[k]; }
    __device__ __forceinline__ void add(int k, const floatx4 &y) { o[k] = o[k] + y; }

    template <bool WIN>
    __device__ __forceinline__ void tile(uint32_t stage, float scale_log2, bool masked, int t0, int lim, int sinks, int low,
                                         uint32_t okbits) {
        const int lane = kq_lane(), c = lane & 15, g = lane >> 4;
        floatx4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        const uint32_t ka = stage + (uint32_t)(c * C::kRow) + 16u * (uint32_t)(C::kswz(c) ^ g);
        pipelined<2 * NQ * C::NP, 6>(
            [&](int x) {
                const int b = x % 2, pl = x / 2 % C::NP, d = x / (2 * C::NP);
                const uint32_t kd = (ka ^ (uint32_t)(16 * ((4 * d) & C::kSw))) + (uint32_t)(16 * ((4 * d) & ~C::kSw));
                return lds_half8(kd + (uint32_t)(pl * C::kPlane + 16 * b * C::kRow));
            },
            [&](int x, const half8_t &f) { s[x % 2] = mfma<BF>(f, qf[x / (2 * C::NP)], s[x % 2]); });
        if (masked) {
            const Shown shown(t0 + 4 * g, lim, sinks, low);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[b][i] = shown.template at<WIN>(16 * b + i) && ((okbits >> b) & 1) ? s[b][i] : -INFINITY;
        }
        float tmax = max3(max3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
        tmax = max_over_groups(max3(max3(tmax, s[1][1], s[1][2]), s[1][3], s[1][3])) * scale_log2;
        const bool up = tmax > m_run + slack<BF>();
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float alpha = up ? __builtin_amdgcn_exp2f(m_run - tmax) : 1.f;
            m_run = up ? tmax : m_run;
            l_part *= alpha;
#pragma unroll
            for (int j = 0; j < NR; ++j) o[j] = o[j] * alpha;
        }
        const float m_use = (m_run == -INFINITY ? 0.f : m_run) - shift<BF, false>();
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], scale_log2, -m_use));
        l_part += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        const half8_t pf = __builtin_bit_cast(half8_t, u32x4{pack2<BF>(p[0], p[1]), pack2<BF>(p[2], p[3]),
                                                             pack2<BF>(p[4], p[5]), pack2<BF>(p[6], p[7])});
        // lane 16 g + i: tokens 4 g + i / 4 (+ 16), values 16 j + 4 (i % 4) ..
        const int tr = 4 * g + ((lane >> 2) & 3);
        const uint32_t va = stage + C::kHalf + (uint32_t)(tr * C::kRow) +
                            16u * (uint32_t)(C::vswz(tr) ^ ((lane >> 1) & 1)) + 8u * (lane & 1);
        pipelined<NR * C::NP, 6>(
            [&](int x) {
                const int j = x % NR, pl = x / NR;
                const uint32_t at = va ^ (uint32_t)(16 * ((2 * j) & C::kSw));
                const uint32_t up = (uint32_t)(16 * ((2 * j) & ~C::kSw) + pl * C::kPlane);
                const u32x2 a = lds_tr(at, up), b = lds_tr(at, up + 16 * C::kRow);
                return __builtin_bit_cast(half8_t, u32x4{a.x, a.y, b.x, b.y});
            },
            [&](int x, const half8_t &f) { o[x % NR] = mfma<BF>(f, pf, o[x % NR]); });
        kq_mfma_drain();
    }
};

// The first halves of two 8-bit values.  fp16's are cut, not rounded: past 65504
// they stay there, and the second halves take the rest.
template <bool BF>
__device__ __forceinline__ uint32_t first_halves(float a, float b) {
    if constexpr (BF) return pack2<BF>(a, b);
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}

template <int D, bool BF, bool Q8, bool WIN>
__device__ __forceinline__ void chunk_work(const PagedArgs &a, uint8_t *smem, int first, int step) {
    using C = Chunk<D, Q8>;
    using State = std::conditional_t<(D > 128), ChunkState16<D, BF, Q8>, ChunkState<D, BF, Q8>>;
    constexpr int COLS = State::COLS;
    static_assert(C::NW * COLS == group_columns(D, Q8), "columns of a workgroup");
    const uint32_t lds = (uint32_t)(uintptr_t)(LDSP(void))smem;
    const auto odd_flag = (volatile LDSP(int))(uintptr_t)(lds + C::kLds);
    const int lane = kq_lane(), c = lane & (COLS - 1);
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    for (int unit = first;; unit += step) {
        int u = unit, b, slot0;
        Row row;
        if (!find_unit<WIN>(a, [&](const Row &x) { return chunk_units<D>(a, x); }, u, b, row, slot0)) return;
        if (!has_slots(a, row, slot0)) continue;
        const int rest = u / a.Hkv, kvh = u - rest * a.Hkv;
        // the tiles with the most keys first
        const int back = rest / row.splits, s = rest - back * row.splits, blk = row.blocks - 1 - back;
        const int col0 = (blk * C::NW + w) * COLS, cols = row.n * a.G;

        // this lane's column; waves past the row's columns only copy
        const int col = col0 + c;
        const bool live = col < cols;
        const int i = live ? col / a.G : row.n - 1, hq = kvh * a.G + (live ? col - i * a.G : 0);
        const auto seen_by = [&](int cl) { return max(row.before + 1 + min(cl, cols - 1) / a.G, 0); };
        const Window win(a, WIN ? seen_by(blk * C::NW * COLS) : 0);
        // keys by number: the row's, or with a window the block's
        const auto keys = [&](int x) { return WIN ? win.keys(min(x, row.kv)) : x; };
        const int seen = live ? keys(min(seen_by(col), row.kv)) : 0x7fffffff;
        const int least = __builtin_amdgcn_readfirstlane(keys(seen_by(col0)));
        const int most = __builtin_amdgcn_readfirstlane(col0 < cols ? keys(min(seen_by(col0 + COLS - 1), row.kv)) : 0);
        const int least_all = __builtin_amdgcn_readfirstlane(keys(seen_by(blk * C::NW * COLS)));
        const int most_all = __builtin_amdgcn_readfirstlane(keys(min(seen_by((blk + 1) * C::NW * COLS - 1), row.kv)));
        // the first key behind the sinks that is in the window of this lane's column, of
        // the wave's first and last, and of the workgroup's last
        int low = 0, low_first = 0, low_last = 0, low_all = 0;
        if constexpr (WIN) {
            low = live ? win.low(a, seen_by(col)) : 0;
            low_first = __builtin_amdgcn_readfirstlane(win.low(a, seen_by(col0)));
            low_last = __builtin_amdgcn_readfirstlane(win.low(a, seen_by(col0 + COLS - 1)));
            low_all = __builtin_amdgcn_readfirstlane(win.low(a, seen_by((blk + 1) * C::NW * COLS - 1)));
        }
        // whether a tile lies between the sinks and a window's first key in part or whole
        const auto left_out = [&](int t0, int first) { return WIN && t0 < first && t0 + C::BN > a.sinks; };
        const int per = few_columns(row.n, a.G, a.few_limit) ? a.rule.tokens(row.span)
                                                : ((row.span + row.splits - 1) / row.splits + C::BN - 1) / C::BN * C::BN;
        const int t_begin = __builtin_amdgcn_readfirstlane(s * per);
        const int t_end = __builtin_amdgcn_readfirstlane(min(most_all, t_begin + per));

        State st;
        st.init();
        // scores are products of the queries with the scale's sign, times its size;
        // instead of 0, which makes a hidden key's -inf NaN, the least number of all
        // (fp32 subnormals are kept here): no product passes 2^-20 with it
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
        const float scale = fmaxf(fabsf(a.scale_log2), 0x1p-149f);
        const uint16_t *qp = a.q + (int64_t)(row.q0 + i) * a.q_stride + (int64_t)hq * D;
#pragma unroll
        for (int d = 0; d < State::NQ; ++d) {
            const u32x4 v = *(const u32x4 *)(qp + State::qd(d));
            st.qf[d] = __builtin_bit_cast(half8_t, live ? v ^ flip : u32x4{0u, 0u, 0u, 0u});
        }

        if (t_end > t_begin) {
            const int32_t *tab = a.table + (int64_t)b * a.table_stride;
            const int sh = a.lps - 4;
            const int c_last = (t_end - 1) >> 4, p_last = (WIN ? win.piece(c_last) : c_last) >> sh;
            PageIds ids;
            bool all_ok;
            if constexpr (WIN) all_ok = ids.start(a, tab, win, t_begin >> 4, c_last, sh);
            else all_ok = ids.start(a, tab, (t_begin >> 4) >> sh, p_last);
            const int64_t h_off = (int64_t)kvh * a.head_stride;
            // Piece y of the RT tokens at a time of the tile at t0 that this
            // wave copies, of K (even waves) or V (odd waves): where it starts
            // in the pool (values) and in a stage.
            constexpr int NY = C::NW == 4 ? C::BN / 32 : 1, RT = 2 * C::BN / (C::NW * NY);
            static_assert(RT == 16 || RT == 8, "within 16 tokens");
            auto piece = [&](int t0, int y, uint32_t &dst) {
                const int t = RT * (C::NW / 2 * y + (w >> 1));
                // (16 tokens past the end are the last ones again: their keys are hidden)
                const int cb = min((t0 + t) >> 4, c_last), ch = WIN ? win.piece(cb) : cb, p = ch >> sh;
                const int id = ids.at(tab, p, p_last);
                dst = (uint32_t)((w & 1) * C::kHalf + t * C::kRow);
                return (int64_t)((uint32_t)id < (uint32_t)a.n_pages ? id : 0) * a.page_stride + h_off +
                       (int64_t)((ch - (p << sh)) * 16 + (t & 15)) * a.tok_stride;
            };
            const auto swizzle = [&](int t) { return w & 1 ? C::vswz(t) : C::kswz(t); };
            const uint8_t *src = (const uint8_t *)(w & 1 ? a.v : a.k);
            // 16-bit pool: straight to LDS.
            auto copy = [&](int t0, uint32_t stage) {
#pragma unroll
                for (int y = 0; y < NY; ++y) {
                    uint32_t dst;
                    const int64_t off = piece(t0, y, dst);
#pragma unroll
                    for (int x = 0; x < C::kCopies; ++x) {
                        const int at = 64 * x + lane, t = at / C::RC, pc = at - t * C::RC;
                        copy16(src + 2 * off, (uint32_t)(t * a.tok_stride + 8 * (pc ^ swizzle(t))) * 2u,
                               stage + dst + 1024u * x);
                    }
                }
            };
            // 8-bit pool: 16 values of a token a lane and load, with their
            // scale and bias, to registers and later to LDS.
            constexpr int NX = Q8 ? RT * D / 1024 : 1;
            u32x4 held[NY][NX];
            uint32_t held_s[NY][NX], held_b[NY][NX], held_at[NY];
            const uint16_t *src_s = w & 1 ? a.vs : a.ks, *src_b = w & 1 ? a.vb : a.kb;
            auto fetch = [&](int t0) {
#pragma unroll
                for (int y = 0; y < NY; ++y) {
                    const int64_t off = piece(t0, y, held_at[y]);
                    const uint8_t *pv = src + off;
                    const uint16_t *ps = src_s + (off >> 6), *pb = src_b + (off >> 6);
#pragma unroll
                    for (int x = 0; x < NX; ++x) {
                        const uint32_t at = 16u * (uint32_t)(64 * x + lane);
                        held[y][x] = *(const u32x4 *)(pv + at);
                        held_s[y][x] = ps[at >> 6];
                        held_b[y][x] = pb[at >> 6];
                    }
                }
            };
            auto put = [&](uint32_t stage) {
#pragma unroll
                for (int y = 0; y < NY; ++y)
#pragma unroll
                    for (int x = 0; x < NX; ++x) {
                        const int at = 16 * (64 * x + lane), t = at / D, pc = (at - t * D) / 8;
                        const int turn = swizzle(t + (RT < 16 ? 8 * (w >> 1 & 1) : 0));
                        const float sc = f16bits_to_f32<BF>(held_s[y][x]), bi = f16bits_to_f32<BF>(held_b[y][x]);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            u32x4 hi, lo;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t two = held[y][x][2 * half + (i >> 1)] >> (16 * (i & 1));
                                const float u = fmaf((float)(two & 0xFFu), sc, bi), v = fmaf((float)((two >> 8) & 0xFFu), sc, bi);
                                hi[i] = first_halves<BF>(u, v);
                                lo[i] = pack2<BF>(u - f16bits_to_f32<BF>(hi[i] & 0xFFFFu), v - f16bits_to_f32<BF>(hi[i] >> 16));
                            }
                            const uint32_t to = stage + held_at[y] + (uint32_t)(t * C::kRow + 16 * ((pc + half) ^ turn));
                            *(LDSP(u32x4))(uintptr_t)to = hi;
                            *(LDSP(u32x4))(uintptr_t)(to + C::kPlane) = lo;
                        }
                    }
            };
            // Bit j: the tile's 16-token piece j lies in a page of the pool.
            auto pages_ok = [&](int t0) {
                uint32_t ok = (1u << (C::BN / 16)) - 1;
                if (!all_ok)
                    for (int j = 0; j < C::BN / 16; ++j)
                        if ((uint32_t)tab[(WIN ? win.piece(min((t0 >> 4) + j, c_last)) : min((t0 >> 4) + j, c_last)) >> sh] >=
                            (uint32_t)a.n_pages)
                            ok &= ~(1u << j);
                return ok;
            };
            // In a tile with hidden keys, the product of a hidden key's value
            // with its probability 0 would be NaN where the value is an
            // infinity or NaN: such values are made 0 in LDS, and where there
            // are any (tiles that say so in odd_flag), what they do to the
            // columns that see them is added from the pool.
            auto clean = [&](uint32_t stage, int t0) {
                uint32_t odd = 0;
                for (uint32_t at = stage + C::kHalf + 16u * threadIdx.x; at < stage + 2 * C::kHalf; at += 16u * 64u * C::NW) {
                    u32x4 v = *(const LDSP(u32x4))(uintptr_t)at;
                    uint32_t here = 0;
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = finite2<BF>(v[x], here);
                    if (here) *(LDSP(u32x4))(uintptr_t)at = v;
                    odd |= here;
                }
                if (odd) *odd_flag = t0 + 1;
                __syncthreads();
            };
            auto add_odd = [&](int t0, int lim) {
#pragma unroll 1
                for (int t = t0; t < min(t0 + C::BN, t_end); ++t) {
                    const int key = WIN ? 16 * win.piece(t >> 4) + (t & 15) : t;
                    const int id = __builtin_amdgcn_readfirstlane(tab[key >> a.lps]);
                    if ((uint32_t)id >= (uint32_t)a.n_pages) continue;
                    const bool sees = t < lim && (!WIN || t < a.sinks || t >= low);
                    const int64_t off = (int64_t)id * a.page_stride + h_off + (int64_t)(key & ((1 << a.lps) - 1)) * a.tok_stride;
#pragma unroll
                    for (int k = 0; k < State::NR; ++k) {
                        const int64_t at = off + State::run_d(k);
                        floatx4 y;
                        if constexpr (Q8) {
                            const float sc = f16bits_to_f32<BF>(a.vs[at >> 6]), bi = f16bits_to_f32<BF>(a.vb[at >> 6]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                // (fp16: infinite from where the halves are, 2^17.  A comparison
                                // with that in its place spilled 24 to 548 bytes a lane.)
                                const float v = fmaf((float)((const uint8_t *)a.v)[at + e], sc, bi) * (BF ? 1.f : 0x1p111f);
                                y[e] = sees && v - v != 0.f ? v : 0.f;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[e] = sees ? odd_part<BF>(((const uint16_t *)a.v)[at + e]) : 0.f;
                        }
                        st.add(k, y);
                        __builtin_amdgcn_sched_barrier(0);  // (few loads at a time: registers)
                    }
                }
            };
            __syncthreads();  // the last unit's reads
            if constexpr (Q8) {
                fetch(t_begin);
                put(lds);
            } else {
                copy(t_begin, lds);
            }
            if (threadIdx.x == 0) *odd_flag = 0;
            uint32_t stage = lds, other = lds + (C::kStages - 1) * C::kStage;
            for (int t0 = t_begin; t0 < t_end; t0 += C::BN) {
                const bool more = t0 + C::BN < t_end;
                // this tile has landed, and every wave is done with the other stage
                if constexpr (Q8) {
                    __syncthreads();
                    if (more) fetch(t0 + C::BN);
                } else {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    if (more) copy(t0 + C::BN, other);
                }
                // uniform over the workgroup
                const bool hidden = !all_ok || t0 + C::BN > min(least_all, t_end) || left_out(t0, low_all);
                if (hidden) clean(stage, t0);
                // (tiles that no column of the wave sees are passed over)
                if (t0 < most && !(WIN && t0 + C::BN <= low_first && t0 >= a.sinks)) {
                    const int lim = min(seen, t_end);
                    const bool masked = !all_ok || t0 + C::BN > min(least, t_end) || left_out(t0, low_last);
                    st.template tile<WIN>(stage, scale, masked, t0, lim, a.sinks, low, masked ? pages_ok(t0) : 0u);
                    if (hidden && *odd_flag == t0 + 1) add_odd(t0, lim);
                }
                if constexpr (Q8) {
                    if constexpr (C::kStages == 1) __syncthreads();
                    if (more) put(other);
                }
                const uint32_t x = stage;
                stage = other;
                other = x;
            }
        }

        const float l = st.sum();
        if (!live) continue;
        const bool whole = row.splits == 1;
        const float mul = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
        uint16_t *op = a.out + (int64_t)(row.q0 + i) * a.out_stride + (int64_t)hq * D;
        const int64_t slot = slot_of(a, row, slot0, i, hq) + s;
        float *pp = a.part + slot * D;
#pragma unroll
        for (int k = 0; k < State::NR; ++k) {
            const int d = State::run_d(k);
            const floatx4 v = st.run(k) * mul;
            if (whole) *(u32x2 *)(op + d) = u32x2{pack2<BF>(v.x, v.y), pack2<BF>(v.z, v.w)};
            else *(floatx4 *)(pp + d) = v;
        }
        if (!whole && lane < COLS) {
            a.ml[2 * slot] = st.m_run;
            a.ml[2 * slot + 1] = l;
        }
    }
}

// Whether rows of few columns run beside chunks in one launch: a chunk of 500
// tokens and seven decode rows 68 us, in two launches 75 (past head dim 128 their
// tiles take more registers than two waves a SIMD can have).
template <int D>
constexpr bool kBeside = D <= 128;

// The first `wave_groups` workgroups take rows of few columns, a wave a unit, the
// others chunks: decode rows, which wait for memory, run beside a prompt
// chunk's products.  (Eight of each kind in turn instead: 68 -> 81 us.)
template <int D, bool BF, bool Q8, bool WIN>
__global__ __launch_bounds__(64 * chunk_waves(D, Q8), D > 256 ? 1 : 2) void kq_paged_kernel(PagedArgs a, int wave_groups) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    if constexpr (kBeside<D>) {
        if ((int)blockIdx.x < wave_groups) {
            constexpr int NW = chunk_waves(D, Q8);
            const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
            wave_work<D, BF, Q8, false, WIN>(a, NW * (int)blockIdx.x + w, NW * wave_groups);
            return;
        }
    }
    chunk_work<D, BF, Q8, WIN>(a, smem, (int)blockIdx.x - wave_groups, (int)gridDim.x - wave_groups);
}

// Scale of a split of maximum ms beside the common maximum m; a split without
// keys holds zeros and counts nothing, one of NaN scores has a NaN sum l.  Splits
// of scale 0 are added like any other: of a NaN or infinite value a token sees, 0
// times it remains, as within a split.
__device__ __forceinline__ float split_scale(float ms, float m) {
    return ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
}

// (Token, query head) of n splits by one workgroup, or of many splits a quarter
// of its outputs by each of four (SL): thread t handles the float4 of outputs 4 q
// .. 4 q + 3 (q = t % Q) for the splits p, p + P, ... (p = t / Q of P parts),
// rescaled to the common maximum; the P sums are added in part order through LDS.
template <int D, bool BF, int SL>
__device__ __forceinline__ void merge_group(const PagedArgs &a, int64_t slot, int n, int slice, uint16_t *out) {
    constexpr int Q = D / 4 / SL, P = 256 / Q;
    __shared__ float red_m[4];
    __shared__ float4 red_acc[P][Q];
    __shared__ float red_l[P];
    const int t = threadIdx.x, q = t % Q, part = t / Q;
    const float *ml = a.ml + 2 * slot;
    const float4 *po = (const float4 *)(a.part + slot * D) + slice * Q + q;
    float m = -INFINITY;
    for (int s = t; s < n; s += 256) m = fmaxf(m, ml[2 * s]);
    // this thread's first splits, in flight beside the maximum's loads
    constexpr int PRE = 4;
    float4 o_pre[PRE];
    float m_pre[PRE], l_pre[PRE];
#pragma unroll
    for (int k = 0; k < PRE; ++k) {
        const int s = min(part + k * P, n - 1);
        m_pre[k] = ml[2 * s];
        l_pre[k] = ml[2 * s + 1];
        o_pre[k] = po[(int64_t)s * (D / 4)];
    }
    m = wave_max(m);
    __syncthreads();  // the last item's reads
    if ((t & 63) == 0) red_m[t >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    if (part < P) {  // (D = 96: the last threads hold no part)
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
        const auto add = [&](float ms, float ls, const float4 &o) {
            const float f = split_scale(ms, m);
            l += f * ls;
            acc.x += f * o.x;
            acc.y += f * o.y;
            acc.z += f * o.z;
            acc.w += f * o.w;
        };
#pragma unroll
        for (int k = 0; k < PRE; ++k)
            if (part + k * P < n) add(m_pre[k], l_pre[k], o_pre[k]);
#pragma unroll 8
        for (int s = part + PRE * P; s < n; s += P) add(ml[2 * s], ml[2 * s + 1], po[(int64_t)s * (D / 4)]);
        red_acc[part][q] = acc;
        if (q == 0) red_l[part] = l;
    }
    __syncthreads();
    if (part == 0) {
        float4 acc = red_acc[0][q];
        float l = red_l[0];
#pragma unroll
        for (int k = 1; k < P; ++k) {
            const float4 o = red_acc[k][q];
            acc.x += o.x;
            acc.y += o.y;
            acc.z += o.z;
            acc.w += o.w;
            l += red_l[k];
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        *(u32x2 *)(out + 4 * (slice * Q + q)) = u32x2{pack2<BF>(acc.x * inv, acc.y * inv), pack2<BF>(acc.z * inv, acc.w * inv)};
    }
}

// The same by one wave, for at most 64 splits, in the same order of sums: lane s
// holds split s's maximum and sum; the first P splits' sums are loaded beside
// them, and before the item ahead of this one is finished.
template <int D, bool BF>
struct WaveMerge {
    static constexpr int P = 256 / (D / 4), V = D > 128 ? 4 : 2, R = D > 256 ? 2 : 1;  // R runs of V values a lane
    typedef float vec __attribute__((ext_vector_type(V)));
    float ms, ls;
    vec o[R][P];

    __device__ __forceinline__ void load(const PagedArgs &a, int64_t slot, int r, int s0, int n) {
        const float *p = a.part + slot * D + min((r * 64 + kq_lane()) * V, D - V);
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (s0 + k < n) o[r][k] = *(const vec *)(p + (int64_t)(s0 + k) * D);
    }
    __device__ __forceinline__ void start(const PagedArgs &a, int64_t slot, int n) {
        const int lane = kq_lane();
        ms = lane < n ? a.ml[2 * (slot + lane)] : -INFINITY;
        ls = lane < n ? a.ml[2 * (slot + lane) + 1] : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) load(a, slot, r, 0, n);
    }
    __device__ __forceinline__ void finish(const PagedArgs &a, int64_t slot, int n, uint16_t *out) {
        const float f = split_scale(ms, wave_max(ms));
        const auto lane_of = [](float v, int s) {
            return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), s));
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            vec acc[P];
            float l[P];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                acc[k] = vec(0.f);
                l[k] = 0.f;
            }
            for (int s0 = 0; s0 < n; s0 += P) {
                if (s0 > 0) load(a, slot, r, s0, n);
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    if (s0 + k >= n) break;
                    const float fs = lane_of(f, s0 + k);
                    l[k] += fs * lane_of(ls, s0 + k);
#pragma unroll
                    for (int x = 0; x < V; ++x) acc[k][x] += fs * o[r][k][x];
                }
            }
#pragma unroll
            for (int k = 1; k < P; ++k) {
                acc[0] = acc[0] + acc[k];
                l[0] += l[k];
            }
            const float inv = l[0] > 0.f || l[0] != l[0] ? 1.f / l[0] : 0.f;
            const int d = (r * 64 + kq_lane()) * V;
            if (d < D) {
#pragma unroll
                for (int x = 0; x < V; x += 2)
                    *(uint32_t *)(out + d + x) = pack2<BF>(acc[0][x] * inv, acc[0][x + 1] * inv);
            }
        }
    }
};

// Workgroups take a token and query head each (direct), or merge_items of a
// row's at a time.  Waves hide each other's loads: one more register than a third of
// a SIMD's at head dim 64, so two waves in place of three, and 1433 tokens of 16 heads
// take 24 us in place of 20.
template <int D, bool BF, bool DIRECT, bool WIN>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 4))) void kq_paged_merge_kernel(PagedArgs a) {
    const auto out = [&](const Row &r, int x) {
        const int i = x / a.Hq;
        return a.out + (int64_t)(r.q0 + i) * a.out_stride + (int64_t)(x - i * a.Hq) * D;
    };
    const auto slot = [&](const Row &r, int slot0, int x) {
        const int i = x / a.Hq;
        return slot_of(a, r, slot0, i, x - i * a.Hq);
    };
    if constexpr (DIRECT) {
        const Row row = lane_row(row_at<WIN>(a, blockIdx.y), 0);
        const int x = blockIdx.x;
        if (row.splits <= 1 || x >= row.n * a.Hq) return;
        if (row.splits > 64) merge_group<D, BF, kSlices>(a, slot(row, 0, x), row.splits, blockIdx.z, out(row, x));
        else if (blockIdx.z == 0) merge_group<D, BF, 1>(a, slot(row, 0, x), row.splits, 0, out(row, x));
        return;
    }
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    for (int item = blockIdx.x;; item += gridDim.x) {
        int u = item, b, slot0;
        Row row;
        if (!find_unit<WIN>(a, [&](const Row &x) { return merge_units(a, x); }, u, b, row, slot0)) return;
        if (!has_slots(a, row, slot0)) continue;
        const int n = row.splits, items = merge_items(n), end = min((u + 1) * items, row.n * a.Hq);
        if (n <= 64) {
            int x = u * items + w;
            if (x >= end) continue;
            WaveMerge<D, BF> now, next;
            now.start(a, slot(row, slot0, x), n);
            for (; x < end; x += 4) {
                if (x + 4 < end) next.start(a, slot(row, slot0, x + 4), n);
                now.finish(a, slot(row, slot0, x), n, out(row, x));
                now = next;
            }
        } else {
            const int x = u / kSlices;
            merge_group<D, BF, kSlices>(a, slot(row, slot0, x), n, u - x * kSlices, out(row, x));
        }
    }
}

struct Grid {
    dim3 waves, merge;   // x == 0: not launched
    int groups;          // workgroups of chunks (0: none)
    int beside;          // waves of rows of few columns beside them
};

template <int D, bool BF, bool Q8, bool WIN>
int launch_form(const PagedArgs &a, const Grid &g, hipStream_t s) {
    if (g.groups) {
        constexpr int lds = Chunk<D, Q8>::kLds + 16;  // (and a flag)
        static_assert(lds <= 160 << 10, "LDS of a CU");
        static OncePerDevice raised;
        int device = -1;
        if (hipGetDevice(&device) != hipSuccess || !raised(device, [] {
                return hipFuncSetAttribute((const void *)kq_paged_kernel<D, BF, Q8, WIN>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           lds) == hipSuccess;
            }))
            return KQ_ERR_LAUNCH_FAILED;
        constexpr int NW = chunk_waves(D, Q8);
        const int beside = kBeside<D> ? (g.beside + NW - 1) / NW : 0;
        hipLaunchKernelGGL((kq_paged_kernel<D, BF, Q8, WIN>), dim3(beside + g.groups), dim3(64 * NW), lds, s, a, beside);
    }
    if constexpr (has_waves(D)) {
        if (g.waves.x && !(kBeside<D> && g.groups)) {
            if (a.direct) hipLaunchKernelGGL((kq_paged_wave_kernel<D, BF, Q8, true, WIN>), g.waves, dim3(64), 0, s, a);
            else hipLaunchKernelGGL((kq_paged_wave_kernel<D, BF, Q8, false, WIN>), g.waves, dim3(64), 0, s, a);
        }
    }
    if (g.merge.x) {
        if (a.direct) hipLaunchKernelGGL((kq_paged_merge_kernel<D, BF, true, WIN>), g.merge, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((kq_paged_merge_kernel<D, BF, false, WIN>), g.merge, dim3(256), 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

template <int D, bool BF>
int launch(const PagedArgs &a, bool q8, const Grid &g, hipStream_t s) {
    if constexpr (D % 64 == 0)
        if (q8) return a.window ? launch_form<D, BF, true, true>(a, g, s) : launch_form<D, BF, true, false>(a, g, s);
    return a.window ? launch_form<D, BF, false, true>(a, g, s) : launch_form<D, BF, false, false>(a, g, s);
}

// Tokens per split of a row of few columns, by its own keys: the lengths of
// decode attention over contiguous caches, which suit pages as they do those.
// Measured on pages of 64 (us; with the rule, and at 64 / 128 / 256 / 512 tokens),
// where that rule's own sweep has no figures, fp16:
//   16 query heads on 2, head dim 256
//     1 row of  1600  13.4   11.7 / 13.5 / 18.9 / 29.8    16  19.4   19.9 / 17.6 / 22.0 / 33.8
//     1 row of  6400  16.2   13.5 / 16.1 / 22.0 / 32.9    16  56.5   63.0 / 56.9 / 53.9 / 48.2
//     1 of     32768  24.2   25.1 / 21.9 / 24.1 / 35.9    16   219    272 /  244 /  220 /  207
//   the same in 8 bits
//     1 row of  1600  17.4   13.7 / 17.7 / 26.7 / 44.4    16  20.8   18.6 / 20.4 / 28.7 / 47.3
//     1 of     32768  30.7   23.3 / 23.4 / 30.7 / 49.5    16   144    210 /  167 /  142 /  120
//   64 query heads on 4, head dim 128
//     1 row of  1600  12.0    8.8 /  9.8 / 12.1 / 16.8    16  17.9   21.6 / 19.2 / 17.1 / 19.5
//     1 of     32768  19.9   26.7 / 22.7 / 19.4 / 20.2    16   219    366 /  283 /  243 /  219
SplitRule wave_rule(int Hq, int Hkv, int D, bool q8) {
    if (const int forced = env_int("GMLX_KQ_SDPA_SPLIT", 0)) return SplitRule{0, 0, 0, 0, (forced + 63) / 64 * 64};
    return row_split_rule(Hq, Hkv, D, q8);
}

// What a call's splits can come to, from the bounds that the host knows.
struct Plan {
    SplitRule rule;
    int few, many;    // the most splits of a row of few columns, of a chunk
    int few_blocks;   // (PagedArgs)
    bool direct;      // (PagedArgs)
    int64_t slots;    // of the workspace
    int slot_stride;  // (PagedArgs)
};

Plan paged_plan(int64_t T, int64_t B, int Hq, int Hkv, int D, int max_q, int max_kv, bool q8, int window, int sinks) {
    Plan p;
    const int G = Hq / Hkv, limit = few_limit(q8), chunk = limit / G + 1;  // tokens of the shortest chunk
    p.rule = wave_rule(Hq, Hkv, D, q8);
    // Through a window of up to kOneLength keys one length for the call's rows, by what
    // it shows at most: then no row has more splits than a full window, and no grid's
    // waves are left without work.  That of 4096 keys past them, since the longer one by
    // the window leaves a few rows to a few long splits.  Wider windows are filled by few
    // rows: each row's own length there, as without one.  us, lengths by row / one by
    // the window / this, 32 query heads on 8, head dim 128, rows of the window or
    // more, then rows of a tenth to half of it:
    //    1024 keys     1 row  11.6 / 11.6 / 11.6,  9.9 / 10.5 / 10.4    64    70 /   70 /   70,  39 /  29 /  29
    //    4100                 16.0 / 15.9 / 14.2, 11.2 / 14.0 / 11.3         276 /  215 /  232,  81 /  68 /  80
    //    8196                 21.7 / 21.4 / 16.2, 11.9 / 19.9 / 11.9         505 /  399 /  463, 155 / 118 / 155
    //   16004                 22.3 / 22.4 / 20.1, 15.1 / 20.3 / 13.9         772 /  773 /  886, 242 / 245 / 234
    //   20004 (this: by row)  23.9 / 23.7 / 23.9, 15.3 / 20.5 / 15.3         971 /  974 /  971, 299 / 284 / 299
    //   32772 (this: by row)  38.7 / 39.0 / 38.7, 20.8 / 20.9 / 20.8        1591 / 1591 / 1591, 452 / 516 / 452
    // and one row of 1800 keys through 32768 or more 12.5 / 19.9 / 12.5, at head dim 256 15.1
    // / 31.6 / 15.1.  Over four head counts and types, 1, 16 and 64 rows, in the geometric
    // mean: up to 3000 keys by row 1.02 of this; 4100 to 16004 by row 1.04, one by the window
    // 1.03; 20004 one 1.00 of this, 32772 1.06.
    constexpr int kOneLength = 16384;
    if (window) {
        const int span = window_span(1 << 30, window, sinks, 1, G, 16);
        if (span <= kOneLength) p.rule = SplitRule{0, 0, 0, 0, p.rule.tokens(span < 4096 ? span : 4096)};
    }
    p.few = chunk > 1 ? most_row_splits(p.rule, max_kv) : 1;
    p.many = max_q >= chunk ? paged_splits(p.rule, chunk, max_kv, G, Hkv, limit, group_columns(D, q8), group_slots(D, q8),
                                           window ? kLeastUnits : 0)
                            : 1;
    const int64_t most = p.few > p.many ? p.few : p.many;
    const int64_t columns = (int64_t)max_q * G < limit ? (int64_t)max_q * G : limit;
    p.few_blocks = (int)(columns + 15) / 16;
    // One slot a token, query head and split, where a token's place gives its
    // slots (by_token); or, where slots follow those of the rows before, tokens of
    // rows of few columns at their splits and the others at a chunk's (by_row).  A
    // chunk has at most group_slots workgroups' columns (splits <= group_slots /
    // workgroups), a row of few columns few_limit a kv head.
    const int64_t tokens = T < B * max_q ? T : B * max_q, few_tokens = tokens < B * (limit / G) ? tokens : B * (limit / G);
    const int64_t rest = p.few < p.many ? tokens : tokens - few_tokens;  // (the more of the two)
    const int64_t chunk_row = (int64_t)group_slots(D, q8) * group_columns(D, q8);
    const int64_t chunks = B < T / chunk ? B : T / chunk;
    const int64_t chunk_slots = rest * Hq * p.many < chunks * chunk_row ? rest * Hq * p.many : chunks * chunk_row;
    const int64_t by_token = T * Hq * most;
    const int64_t by_row = (p.few > 1 ? few_tokens * Hq * p.few : 0) + (p.many > 1 ? chunk_slots : 0);
    // Direct grids need the first; where padding makes it more than any rows could
    // take, they are not worth its memory.
    const int64_t few_row = (int64_t)limit * Hkv * p.few, many_row = p.many > 1 ? chunk_row : 0;
    const int64_t waves = (int64_t)p.few * p.few_blocks * Hkv * B, items = (max_q < T ? max_q : T) * Hq;
    p.direct = B < (1 << 16) && waves <= kDirect && items * B <= kDirect &&
               (most < 2 || by_token <= B * (few_row > many_row ? few_row : many_row));
    p.slots = most < 2 ? 0 : p.direct || by_token < by_row ? by_token : by_row;
    p.slot_stride = most > 1 && p.slots == by_token ? (int)most : 0;
    return p;
}

// 31-bit numbers of tokens and heads, and of keys (a split past the last among them).
bool sizes_fit(int64_t T, int64_t B, int Hq, int max_kv) { return T * Hq <= (1 << 30) && B <= (1 << 20) && max_kv <= (1 << 30); }

size_t part_bytes(int64_t slots, int D) { return ((size_t)slots * D * 4 + 255) & ~(size_t)255; }

// Whether 32-bit numbers count a call's partials and units (a grid's step past
// the last of them too).  Units of the two kernels apart, since a chunk of many
// columns has few splits however many keys it has: blocks times splits of a row
// come to group_slots / Hkv, or to its blocks alone.
bool numbers_fit(const Plan &p, int64_t T, int64_t B, int Hq, int Hkv, int D, bool q8) {
    constexpr int64_t kMost = ((int64_t)1 << 31) - (1 << 17);
    if (p.slots >= (int64_t)1 << 31) return false;
    const int G = Hq / Hkv, limit = few_limit(q8), cols = group_columns(D, q8);
    const int64_t rows = T < B ? T : B;
    const int few_blocks = has_waves(D) ? (limit + 15) / 16 : 1;
    const int64_t few = G <= limit ? rows * few_blocks * Hkv * p.few : 0;
    const int64_t many = rows * group_slots(D, q8) + (T * G / cols + rows) * Hkv;
    return has_waves(D) ? few < kMost && many < kMost : few + many < kMost;
}

// (31-bit numbers of keys)
bool window_fits(int32_t window, int32_t sinks) {
    return window >= 1 && window <= (1 << 30) && sinks >= 0 && sinks <= (1 << 30);
}

// The most keys that a row's splits divide (window 0: none).
int most_span(int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q, int32_t max_kv, bool q8, int32_t window, int32_t sinks) {
    return window ? window_span(max_kv, window, sinks, max_q, Hq / Hkv, group_columns(D, q8)) : max_kv;
}

size_t workspace_bytes_of(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q, int32_t max_kv, int q8,
                          int32_t window, int32_t sinks) {
    if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hkv > 1024 || D <= 0 || max_q <= 0 || max_kv <= 0 ||
        !sizes_fit(T, B, Hq, max_kv))
        return 0;
    const int span = most_span(Hq, Hkv, D, max_q, max_kv, q8 != 0, window, sinks);
    const Plan p = paged_plan(T, B, Hq, Hkv, D, max_q, span, q8 != 0, window, sinks);
    return p.slots && numbers_fit(p, T, B, Hq, Hkv, D, q8 != 0) ? part_bytes(p.slots, D) + (size_t)p.slots * 8 : 0;
}

int attend(const void *q, int64_t q_stride, const kq_paged_pool *pool, const int32_t *block_table, int64_t table_stride,
           int32_t table_width, const int32_t *kv_lens, const int32_t *cu_q, int32_t T, int32_t B, int32_t Hq, int32_t max_q,
           int32_t max_kv, int32_t window, int32_t sinks, float scale, void *out, int64_t out_stride, void *workspace,
           size_t workspace_bytes, kq_stream_t stream) {
    if (const int rc = kq_pool_check(pool)) return rc;
    if (T == 0 || B == 0) return KQ_OK;
    if (!q || !block_table || !kv_lens || !cu_q || !out) return KQ_ERR_NULL_POINTER;
    const int Hkv = pool->Hkv, D = pool->D;
    if (T < 0 || B < 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 64 || max_q < 1 || max_kv < 1 ||
        table_width < 1 || table_stride < table_width)
        return KQ_ERR_BAD_SHAPE;
    // (in the kernels' log2 units, too)
    if (!(fabsf(scale * 1.4426950408889634f) <= 3.4028235e38f)) return KQ_ERR_BAD_ARGUMENT;
    if (!sizes_fit(T, B, Hq, max_kv) || q_stride < (int64_t)Hq * D || out_stride < (int64_t)Hq * D) return KQ_ERR_BAD_SHAPE;
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_stride | out_stride) & 7)) return KQ_ERR_BAD_ALIGN;
    const int span = most_span(Hq, Hkv, D, max_q, max_kv, pool->k_scales != nullptr, window, sinks);
    const Plan plan = paged_plan(T, B, Hq, Hkv, D, max_q, span, pool->k_scales != nullptr, window, sinks);
    const int64_t most = plan.few > plan.many ? plan.few : plan.many;
    if (!numbers_fit(plan, T, B, Hq, Hkv, D, pool->k_scales != nullptr)) return KQ_ERR_BAD_SHAPE;
    const size_t need = plan.slots ? part_bytes(plan.slots, D) + (size_t)plan.slots * 8 : 0;
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
    a.group_cols = group_columns(D, a.ks != nullptr);
    a.group_slots = group_slots(D, a.ks != nullptr);
    a.few_limit = few_limit(a.ks != nullptr);
    a.few_cols = has_waves(D) ? 16 : a.group_cols;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.window = window;
    a.sinks = sinks;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.part = (float *)workspace;
    a.ml = (float *)((char *)workspace + part_bytes(plan.slots, D));
    a.rule = plan.rule;
    a.slot_stride = plan.slot_stride;
    a.slots = (int32_t)plan.slots;
    a.few_blocks = plan.few_blocks;
    a.direct = plan.direct;
    // Bounds of the units; past them the grids' waves and workgroups take the
    // rest in turn.  Where a wave or workgroup for every unit that the longest
    // rows would have is no large grid, each finds its own from its place there;
    // else they sum over the rows' units.
    Grid g;
    const int64_t rows = T < B ? T : B, items = (int64_t)(max_q < T ? max_q : T) * Hq;
    g.waves = g.merge = dim3(0);
    const int64_t blocks = (((int64_t)T * a.G + a.group_cols - 1) / a.group_cols + rows) * Hkv;
    int64_t many = blocks * (has_waves(D) ? plan.many : most);
    if (has_waves(D)) {
        // A chunk's splits times its blocks are no more than group_slots, or it has one:
        // without this bound workgroups that find no unit queue up behind the others (us,
        // without / with it: 4096 tokens alone 175 / 167, in 8 bits 327 / 307, four rows
        // of 1000 over 5000 386 / 371, 2048 through a window of 2000 99 / 93; 2048 behind
        // 6000 276 / 276).
        const int64_t filled = rows * a.group_slots + (blocks > a.group_slots ? blocks - a.group_slots : 0);
        many = many < filled ? many : filled;
    }
    g.groups = has_waves(D) && few_columns(max_q, a.G, a.few_limit) ? 0 : (int)(many < (1 << 14) ? many : (1 << 14));
    g.beside = 0;
    if (has_waves(D) && a.G <= a.few_limit) {
        const int64_t n = rows * Hkv * plan.few * a.few_blocks;
        if (a.direct) g.waves = dim3(a.few_blocks > 1 ? (plan.few + 7) / 8 * 16 : plan.few, Hkv, B);
        else g.waves = dim3((unsigned)(n < (1 << 16) ? n : (1 << 16)));
        if (g.groups) g.beside = (int)(n < (1 << 13) ? n : (1 << 13));
    }
    if (plan.slots) {
        const int64_t n = most > 64 ? kSlices * items * B : most > 8 ? items * B : (int64_t)T * Hq / 16 + B;
        g.merge = a.direct ? dim3((unsigned)items, B, most > 64 ? kSlices : 1) : dim3((unsigned)(n < kMergeGroups ? n : kMergeGroups));
    }
    const bool q8 = a.ks != nullptr, bf = pool->dtype == KQ_DTYPE_BF16;
    hipStream_t s = (hipStream_t)stream;
    switch (D) {
    case 64: return bf ? launch<64, true>(a, q8, g, s) : launch<64, false>(a, q8, g, s);
    case 96: return bf ? launch<96, true>(a, q8, g, s) : launch<96, false>(a, q8, g, s);
    case 128: return bf ? launch<128, true>(a, q8, g, s) : launch<128, false>(a, q8, g, s);
    case 256: return bf ? launch<256, true>(a, q8, g, s) : launch<256, false>(a, q8, g, s);
    default: return bf ? launch<512, true>(a, q8, g, s) : launch<512, false>(a, q8, g, s);
    }
}

}  // namespace

extern "C" {

size_t kq_sdpa_paged_workspace_bytes(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q,
                                     int32_t max_kv, int q8) {
    return workspace_bytes_of(T, B, Hq, Hkv, D, max_q, max_kv, q8, 0, 0);
}

int kq_sdpa_paged(const void *q, int64_t q_stride, const kq_paged_pool *pool, const int32_t *block_table,
                  int64_t table_stride, int32_t table_width, const int32_t *kv_lens, const int32_t *cu_q, int32_t T,
                  int32_t B, int32_t Hq, int32_t max_q, int32_t max_kv, float scale, void *out, int64_t out_stride,
                  void *workspace, size_t workspace_bytes, kq_stream_t stream) {
    return attend(q, q_stride, pool, block_table, table_stride, table_width, kv_lens, cu_q, T, B, Hq, max_q, max_kv, 0, 0,
                  scale, out, out_stride, workspace, workspace_bytes, stream);
}

size_t kq_sdpa_paged_window_workspace_bytes(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_q,
                                            int32_t max_kv, int q8, int32_t window, int32_t sinks) {
    if (!window_fits(window, sinks)) return 0;
    return workspace_bytes_of(T, B, Hq, Hkv, D, max_q, max_kv, q8, window, sinks);
}

int kq_sdpa_paged_window(const void *q, int64_t q_stride, const kq_paged_pool *pool, const int32_t *block_table,
                         int64_t table_stride, int32_t table_width, const int32_t *kv_lens, const int32_t *cu_q, int32_t T,
                         int32_t B, int32_t Hq, int32_t max_q, int32_t max_kv, int32_t window, int32_t sinks, float scale,
                         void *out, int64_t out_stride, void *workspace, size_t workspace_bytes, kq_stream_t stream) {
    if (!window_fits(window, sinks)) return KQ_ERR_BAD_SHAPE;
    return attend(q, q_stride, pool, block_table, table_stride, table_width, kv_lens, cu_q, T, B, Hq, max_q, max_kv, window,
                  sinks, scale, out, out_stride, workspace, workspace_bytes, stream);
}

}  // extern "C"
