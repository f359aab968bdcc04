// Drafted tokens checked against the target's logits (kq_verify_drafts).
//
// Row t of the logits at temperature c has the weights
//   e_v = exp((x_v - max x) / c), p_v = e_v / Z, Z = sum of e_v.
// The draft d behind it stands where u q_d Z < e_d (u q_d < p_d), q the
// probabilities that it was drawn from, or 1 for d alone.  Behind the first draft of
// a row that does not stand, or behind all of them, comes the token v at which
// the running sum of w passes r times the whole: w = max(e - q Z, 0) (e without e_d
// where d alone was proposed) behind a refused draft, e behind the last.
//
// A running sum over V tokens has V borders that r may fall next to, so weights
// (good to 4 10^-14) and sums are fp64, where fp32's 10^-7 would put one draw in a
// hundred on the other side of some border at V = 10^5.  So is a temperature given
// as a number: 0.7 rounded to fp32 alone, off by 1.7 10^-8, moved 16 of 60000 draws
// at V = 152064.
#include <algorithm>

#include "kq_attn.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// What a slice of a logits row comes to.
struct Part {
    float m;     // its largest value, -infinity: none
    int32_t at;  // the lowest token that has it
    double sum;  // of exp((x - m) / c)
};

struct VerifyArgs {
    const void *logits, *probs;
    int64_t stride, probs_stride;
    const int32_t *tokens, *cu, *kv;
    const float *u, *draws, *temps;
    double rate;  // log2(e) / c without temps, 0 at a temperature of 0
    int32_t T, B, V, S;  // S: slices a row
    int32_t probs_type;
    Part *part;    // [T][S]
    double *rest;  // [B][S]: sums of max(e - q Z, 0)
    struct Verdict *verdict;  // [B], NULL: found by the last kernel
    int32_t decides;  // the rest's kernel finds the verdicts
    int32_t *accepted, *next, *keep;
};

// 2^y for y <= 0 as p 2^n: a polynomial of y's distance to the nearest whole number,
// within 4 10^-14 and exact at 0, with n put in the exponent of 1.  (From a table of
// 64 or 256 powers in LDS and a polynomial of the fourth or third power, 397 rows of
// 152064 values took 58 and 62 us, with this one 56: the table's bank conflicts
// cost more than five fp64 steps.)  Below 2^-1000 (and of NaN) 2^-1000, which no sum
// beside a largest weight of 1 notices.
struct Power {
    double scale, p;  // their product
};
__device__ __forceinline__ Power power(double y) {
    constexpr double kRound = 0x1.8p52;  // its unit is 1: adding it rounds, the integer in the low bits
    y = fmax(y, -1000.0);
    const double t = y + kRound, r = y - (t - kRound);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    // least maximum of the error, the constant term 1
    double p = fma(r, 1.0203121063391729e-07, 1.3255224878668817e-06);
    p = fma(r, p, 1.525268684626772e-05);
    p = fma(r, p, 0.00015403455852453838);
    p = fma(r, p, 0.0013333558179043112);
    p = fma(r, p, 0.009618129159402558);
    p = fma(r, p, 0.055504108664760424);
    p = fma(r, p, 0.2402265069581299);
    p = fma(r, p, 0.6931471805599453);
    p = fma(r, p, 1.0);
    return Power{__builtin_bit_cast(double, (uint64_t)((n + 1023u) << 20) << 32), p};
}

// Values of 16 bytes of logits.
template <int DT>
constexpr int kValues = DT == KQ_DTYPE_F32 ? 4 : 8;

template <int DT>
__device__ __forceinline__ float value(const void *p, int64_t i) {
    if constexpr (DT == KQ_DTYPE_F32) return ((const float *)p)[i];
    else return f16bits_to_f32<DT == KQ_DTYPE_BF16>(((const uint16_t *)p)[i]);
}

// Values i .. i + N - 1 of a row of V (rows start at any multiple of a value's
// size); `past` for those behind its end.
template <int DT, int N>
__device__ __forceinline__ void values(const void *row, int i, int V, float past, float (&x)[N]) {
    if (i <= V - N) {
        if constexpr (DT == KQ_DTYPE_F32) {
            typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const vec w = *(const vec *)((const float *)row + i + j);
                x[j] = w.x, x[j + 1] = w.y, x[j + 2] = w.z, x[j + 3] = w.w;
            }
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(N / 2), aligned(2)));
            const vec w = *(const vec *)((const uint16_t *)row + i);
#pragma unroll
            for (int j = 0; j < N; ++j)
                x[j] = f16bits_to_f32<DT == KQ_DTYPE_BF16>((w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = i < V - j ? value<DT>(row, i + j) : past;
    }
}

// A logit as it counts: NaN as -infinity, +infinity as the largest number.  (A
// weight of either is right as it is.)
__device__ __forceinline__ float counted(float x) { return x != x ? -INFINITY : fminf(x, 3.4028235e38f); }

__device__ __forceinline__ bool greedy(const VerifyArgs &a, int b) { return a.temps ? !(a.temps[b] > 0.f) : a.rate == 0.0; }

// log2(e) / c of row b.
__host__ __device__ __forceinline__ double rate_at(double c) { return 1.4426950408889634074 / c; }
__device__ __forceinline__ double rate_of(const VerifyArgs &a, int b) {
    return a.temps ? rate_at(fminf(a.temps[b], 3.4028235e38f)) : a.rate;
}

// The weight of x <= m (both fp64 steps are exact for x = m), and the same, 0 below 2^-1000.
__device__ __forceinline__ double weight(float x, float m, double rate) {
    const Power e = power(((double)x - (double)m) * rate);
    return e.scale * e.p;
}
__device__ __forceinline__ double weight0(float x, float m, double rate) {
    return weight(x, m, rate) - 0x1p-1000;
}

// Infinities among a thread's values as the largest number, where that is m (NaN
// stays, and weighs nothing).
template <int N>
__device__ __forceinline__ void cap(float m, float (&x)[N]) {
    if (m < 3.4028235e38f) return;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = x[j] > 3.4028235e38f ? 3.4028235e38f : x[j];
}

// v of another lane of the wave (a DPP pattern), or `none` where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ float from_lane(float v, float none) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL,
                                                                 ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lane(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double of_lane(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, from_lane<0x111, 0xf>(v, -INFINITY));  // row_shr:1, 2, 4, 8
    v = fmaxf(v, from_lane<0x112, 0xf>(v, -INFINITY));
    v = fmaxf(v, from_lane<0x114, 0xf>(v, -INFINITY));
    v = fmaxf(v, from_lane<0x118, 0xf>(v, -INFINITY));
    v = fmaxf(v, from_lane<0x142, 0xa>(v, -INFINITY));  // row_bcast:15, 31
    v = fmaxf(v, from_lane<0x143, 0xc>(v, -INFINITY));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// Inclusive running sum over the wave's lanes, and the whole sum.
__device__ __forceinline__ double wave_scan(double v) {
    v += from_lane<0x111, 0xf>(v);
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);
    v += from_lane<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) { return of_lane(wave_scan(v), 63); }

// The larger of two (value, token), the lower token of equal values.
__device__ __forceinline__ void take_larger(float &m, int &at, float m2, int at2) {
    const bool other = m2 > m || (m2 == m && at2 < at);
    m = other ? m2 : m;
    at = other ? at2 : at;
}
__device__ __forceinline__ void wave_largest(float &m, int &at) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off);
        const int at2 = __shfl_xor(at, off);
        take_larger(m, at, m2, at2);
    }
}

// The row b that logits row t belongs to: the last whose first row is at or before
// t (rows without logits are passed over).
__device__ __forceinline__ int row_at(const int32_t *cu, int B, int t) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A slice: 256 times 16 bytes of a row, kChunks of them a lane to the wave that sums
// it, one a thread to the workgroup that looks for a token in it.
constexpr int kChunks = kThreads / 64;

// One slice of one logits row a wave, held in registers between the maximum and the
// sum, so the logits are read once; waves share nothing, so that some load while
// others calculate (a slice four times as long by a workgroup together:
// 57 us; the next kernels look through four times as many tokens then).
template <int DT>
__global__ __launch_bounds__(kThreads) void kq_verify_rows_kernel(VerifyArgs a) {
    constexpr int N = kValues<DT>;
    const int lane = kq_lane(), unit = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const int t = unit / a.S, s = unit - t * a.S;
    if (t >= min(a.cu[a.B], a.T)) return;
    const uint8_t *row = (const uint8_t *)a.logits + (int64_t)t * a.stride * (16 / N);
    float x[kChunks][N];
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
        values<DT, N>(row, min(((s * kChunks + c) * 64 + lane) * N, a.V), a.V, -INFINITY, x[c]);
    const int b = a.temps ? row_at(a.cu, a.B, t) : 0;
    float m = -INFINITY;
    int at = 0x7fffffff;
    double sum = 0.0;
    if (greedy(a, b)) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float v = counted(x[c][j]);
                if (v > m) {
                    m = v;
                    at = ((s * kChunks + c) * 64 + lane) * N + j;
                }
            }
        wave_largest(m, at);
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) m = fmaxf(m, x[c][j]);  // (drops NaN)
        m = fminf(wave_max(m), 3.4028235e38f);
        if (m > -INFINITY) {
            const double rate = rate_of(a, b);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                cap(m, x[c]);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const Power e = power(((double)x[c][j] - (double)m) * rate);
                    sum = fma(e.scale, e.p, sum);
                }
            }
            sum = wave_sum(sum);
        }
    }
    if (lane == 0) a.part[(int64_t)t * a.S + s] = Part{m, at, sum};
}

// Where row b ends, the same in every thread.
struct Verdict {
    double Z;
    int t;         // the logits row whose token follows
    int accepted;  // drafts that stand
    int draft;     // the refused one, -1: none was, or it is no token
    float m;       // its largest logit, -infinity: none
    int top;       // the lowest token that has it (greedy)
};

template <int PT>
__device__ __forceinline__ double prob(const void *probs, int64_t at) {
    return fmax((double)value<PT>(probs, at), 0.0);  // (NaN: 0)
}

__device__ __forceinline__ double prob_at(const VerifyArgs &a, int t, int v) {
    const int64_t at = (int64_t)t * a.probs_stride + v;
    return a.probs_type == KQ_DTYPE_F32    ? prob<KQ_DTYPE_F32>(a.probs, at)
           : a.probs_type == KQ_DTYPE_BF16 ? prob<KQ_DTYPE_BF16>(a.probs, at)
                                           : prob<KQ_DTYPE_F16>(a.probs, at);
}

// A wave a draft, kWaves of them at a time until one does not stand.  n > 0.
template <int DT>
__device__ __forceinline__ Verdict decide(const VerifyArgs &a, int b, int q0, int n) {
    __shared__ float s_m[kWaves];
    __shared__ int s_top[kWaves], s_ok[kWaves], s_d[kWaves];
    __shared__ double s_z[kWaves];
    const int lane = kq_lane(), w = threadIdx.x >> 6;
    const bool pick_top = greedy(a, b);
    const double rate = rate_of(a, b);
    for (int i0 = 0;; i0 += kWaves) {
        const int i = min(i0 + w, n - 1), t = q0 + i;
        const Part *part = a.part + (int64_t)t * a.S;
        const bool last = i == n - 1;
        const int d = last ? -1 : a.tokens[t + 1];
        const bool known = d >= 0 && d < a.V;
        const float x = known ? counted(value<DT>(a.logits, (int64_t)t * a.stride + d)) : -INFINITY;
        const double q = known && !pick_top && a.probs ? prob_at(a, t, d) : 1.0;
        float m = -INFINITY;
        int at = 0x7fffffff;
        double z = 0.0;
        bool ok;
        if (pick_top) {
            for (int s = lane; s < a.S; s += 64) take_larger(m, at, part[s].m, part[s].at);
            wave_largest(m, at);
            ok = known && d == at;
        } else {
            const float u = last ? 0.f : a.u[t];
            const Part first = lane < a.S ? part[lane] : Part{-INFINITY, 0, 0.0};
            m = first.m;
            for (int s = lane + 64; s < a.S; s += 64) m = fmaxf(m, part[s].m);
            m = wave_max(m);
            if (m > -INFINITY) {
                z = first.sum * weight(first.m, m, rate);
                for (int s = lane + 64; s < a.S; s += 64) z += part[s].sum * weight(part[s].m, m, rate);
            }
            z = wave_sum(z);
            ok = known && x > -INFINITY && (double)u * q * z < weight0(x, m, rate);
        }
        __syncthreads();  // the last round's reads
        if (lane == 0) {
            s_m[w] = m;
            s_d[w] = known ? d : -1;
            s_top[w] = at;
            s_z[w] = z;
            s_ok[w] = ok && !last;
        }
        __syncthreads();
        int k = 0;
        while (k < kWaves && s_ok[k]) ++k;
        if (k < kWaves) {
            // (waves past the row's end repeat its last row, which is never a draft)
            const int j = min(i0 + k, n - 1);
            return Verdict{s_z[k], q0 + j, j, s_d[k], s_m[k], pick_top ? s_top[k] : 0};
        }
    }
}

__device__ __forceinline__ bool row_of(const VerifyArgs &a, int b, int &q0, int &n) {
    q0 = min(max(a.cu[b], 0), a.T);
    n = min(max(a.cu[b + 1], q0), a.T) - q0;
    return n > 0;
}

// max(e - q Z, 0) of N tokens from i on; 0 past the end.
template <int DT, int PT, int N>
__device__ __forceinline__ void rest_of(const VerifyArgs &a, const Verdict &r, double rate, int i,
                                        double (&w)[N]) {
    float x[N], q[N];
    values<DT, N>((const uint8_t *)a.logits + (int64_t)r.t * a.stride * (DT == KQ_DTYPE_F32 ? 4 : 2), i, a.V, -INFINITY, x);
    values<PT, N>((const uint8_t *)a.probs + (int64_t)r.t * a.probs_stride * (PT == KQ_DTYPE_F32 ? 4 : 2), i, a.V, 0.f, q);
    cap(r.m, x);
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = fmax(weight0(x[j], r.m, rate) - fmax((double)q[j], 0.0) * r.Z, 0.0);
}

// Where each row ends, one workgroup a row.
template <int DT>
__global__ __launch_bounds__(kThreads) void kq_verify_decide_kernel(VerifyArgs a) {
    const int b = blockIdx.x;
    int q0, n;
    if (!row_of(a, b, q0, n)) return;
    const Verdict r = decide<DT>(a, b, q0, n);
    if (threadIdx.x == 0) a.verdict[b] = r;
}

// The sum of max(e - q Z, 0) over a slice, by a wave.
template <int DT, int PT>
__device__ __forceinline__ double rest_sum(const VerifyArgs &a, const Verdict &r, double rate, int s) {
    constexpr int N = kValues<DT>;
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        double w[N];
        rest_of<DT, PT, N>(a, r, rate, min(((s * kChunks + c) * 64 + kq_lane()) * N, a.V), w);
#pragma unroll
        for (int j = 0; j < N; ++j) sum += w[j];
    }
    return wave_sum(sum);
}

// These sums of every slice, a wave each, of rows whose draft was refused.  decides:
// every workgroup finds for itself where its row ends.
template <int DT, int PT>
__global__ __launch_bounds__(kThreads) void kq_verify_rest_kernel(VerifyArgs a) {
    const int b = blockIdx.y, s = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    int q0, n;
    if (!row_of(a, b, q0, n)) return;
    const Verdict r = a.decides ? decide<DT>(a, b, q0, n) : a.verdict[b];
    if (a.decides && blockIdx.x == 0 && threadIdx.x == 0) a.verdict[b] = r;
    if (s >= a.S || r.accepted == n - 1 || greedy(a, b) || !(r.m > -INFINITY)) return;
    const double sum = rest_sum<DT, PT>(a, r, rate_of(a, b), s);
    if (kq_lane() == 0) a.rest[(int64_t)b * a.S + s] = sum;
}

// The most slices of a row whose last kernel sums the rest beside q itself, two
// rounds of its waves, in place of a launch before it (us behind the rows' kernel,
// 128 rows of 4 drafts: 4 slices 15 in place of 18, 8 19.5 in place of 18.5 and that
// launch, 12 23 in place of 19, 15 27 in place of 19).
constexpr int kFewSlices = 8;
// The most workgroups of the rest's kernel that find their rows' ends each, in
// place of a launch (us, rows of 64 slices, 4 drafts: 1 row 4.7 in place of 3.7 and
// 2.3, 48 11.7 in place of 4.9 and 9.5, 96 16.5 in place of 5.3 and 12.7; 128, 2048
// workgroups, 20.6 in place of 5.2 and 15.0, 160 24.7 in place of 5.2 and 16.6).
constexpr int kDecide = 1536;

// The token that follows, one workgroup a row: the slice whose running sum passes
// r times the whole, then the token within it.
template <int DT, int PT>
__global__ __launch_bounds__(kThreads) void kq_verify_pick_kernel(VerifyArgs a) {
    constexpr int N = kValues<DT>;
    __shared__ double red[kWaves], s_rest[kFewSlices];
    __shared__ double s_target;
    __shared__ int s_how, s_slice, s_first, s_last;
    const int b = blockIdx.x, lane = kq_lane(), wv = threadIdx.x >> 6;
    int q0, n;
    if (!row_of(a, b, q0, n)) {
        if (threadIdx.x == 0) {
            a.accepted[b] = 0;
            a.next[b] = -1;
            if (a.keep) a.keep[b] = max(a.kv[b], 0);
        }
        return;
    }
    const Verdict r = a.verdict ? a.verdict[b] : decide<DT>(a, b, q0, n);
    const auto finish = [&](int token) {
        a.accepted[b] = r.accepted;
        a.next[b] = token;
        if (a.keep) a.keep[b] = max(a.kv[b] - (n - 1 - r.accepted), 0);
    };
    const bool none = !(r.m > -INFINITY);
    if (greedy(a, b) || none) {
        if (threadIdx.x == 0) finish(none ? -1 : r.top);
        return;
    }
    const double rate = rate_of(a, b);
    const Part *part = a.part + (int64_t)r.t * a.S;
    const bool refused = r.accepted < n - 1, lone = refused && !a.probs && r.draft >= 0;
    // a thread's weights in a slice: how 0 as they are, 1 without the draft, 2 beside q
    double w[N];
    const auto weigh = [&](int how, int s) {
        const int i = (s * kThreads + (int)threadIdx.x) * N, from = min(i, a.V);
        if (how == 2) {
            rest_of<DT, PT, N>(a, r, rate, from, w);
        } else {
            float x[N];
            values<DT, N>((const uint8_t *)a.logits + (int64_t)r.t * a.stride * (16 / N), from, a.V, -INFINITY, x);
            cap(r.m, x);
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = how == 1 && i + j == r.draft ? 0.0 : weight0(x[j], r.m, rate);
        }
    };
    // A lone draft's slice is summed again without it: taken off the slice's sum, what is
    // left would keep that sum's error, up to all of its digits (10.8 us in place of 11.4,
    // 16 rows of 64 slices; only where the draft holds half of the slice or more 12.3).
    const int own = lone ? r.draft / (kThreads * N) : -1;
    double without = 0.0;
    if (lone) {
        weigh(1, own);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) sum += w[j];
        sum = wave_sum(sum);
        if (lane == 0) red[wv] = sum;
        __syncthreads();
        for (int k = 0; k < kWaves; ++k) without += red[k];
        __syncthreads();
    }
    // wave 0: the slices' running sums
    int how = lone ? 1 : refused && a.probs ? 2 : 0;
    if (how == 2 && !a.verdict) {
        for (int s = wv; s < a.S; s += kWaves) {
            const double sum = rest_sum<DT, PT>(a, r, rate, s);
            if (lane == 0) s_rest[s] = sum;
        }
        __syncthreads();
    }
    if (wv == 0) {
        const auto slice_sum = [&](int s) {
            if (s >= a.S) return 0.0;
            return how == 2 ? (a.verdict ? a.rest[(int64_t)b * a.S + s] : s_rest[s])
                   : s == own && how == 1 ? without
                                          : part[s].sum * weight0(part[s].m, r.m, rate);
        };
        double all = 0.0, first = 0.0;  // (first: this lane's of the first 64)
        for (int pass = 0; pass < 2; ++pass) {
            first = all = slice_sum(lane);
            for (int s = lane + 64; s < a.S; s += 64) all += slice_sum(s);
            all = wave_sum(all);
            if (all > 0.0) break;
            how = 0;  // nothing is left beside q: the target's own
        }
        const float draw = a.draws[b];
        const double target = (draw > 0.f ? (double)draw : 0.0) * all;
        double before = 0.0, at_before = 0.0;
        int slice = 0;
        for (int s0 = 0; s0 < a.S; s0 += 64) {
            const double mine = s0 ? slice_sum(s0 + lane) : first;
            const double run = wave_scan(mine);
            const uint64_t over = __ballot(mine > 0.0 && before + run > target), some = __ballot(mine > 0.0);
            // (none passes a draw of 1: the last slice that has any weight)
            const int pick = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
            if (pick >= 0) {
                slice = s0 + pick;
                at_before = before + of_lane(run, pick) - of_lane(mine, pick);
            }
            if (over) break;
            before += of_lane(run, 63);
        }
        if (lane == 0) {
            s_how = how;
            s_slice = slice;
            s_target = target - at_before;
            s_first = 0x7fffffff;
            s_last = -1;
        }
    }
    __syncthreads();
    const int slice = s_slice;
    const double target = s_target;
    weigh(s_how, slice);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += w[j];
    const double up = wave_scan(sum);
    if (lane == 63) red[wv] = up;
    __syncthreads();
    double run = up - sum;
    for (int k = 0; k < wv; ++k) run += red[k];
    int first = 0x7fffffff, last = -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        run += w[j];
        if (w[j] > 0.0) {
            last = (slice * kThreads + (int)threadIdx.x) * N + j;
            if (first == 0x7fffffff && run > target) first = last;
        }
    }
    if (first != 0x7fffffff) atomicMin(&s_first, first);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (threadIdx.x == 0) finish(s_first != 0x7fffffff ? s_first : s_last);
}

int slices(int V, int dtype) {
    const int len = kThreads * (dtype == KQ_DTYPE_F32 ? 4 : 8);
    return (int)(((int64_t)V + len - 1) / len);
}
size_t part_bytes(int64_t T, int S) { return ((size_t)T * S * sizeof(Part) + 255) & ~(size_t)255; }
size_t need_bytes(int64_t T, int64_t B, int S, bool probs) {
    return part_bytes(T, S) + (probs ? (size_t)B * (S * sizeof(double) + sizeof(Verdict)) : 0);
}

// Grids of fewer than 2^32 threads, and 31-bit numbers of tokens a slice past the last.
bool sizes_fit(int64_t T, int64_t B, int V, int S) {
    return T <= 1 << 22 && B < 1 << 16 && V <= 1 << 28 && T * S <= 1 << 24;
}

template <int DT, int PT>
void launch(const VerifyArgs &a, hipStream_t s) {
    if (a.T) hipLaunchKernelGGL((kq_verify_rows_kernel<DT>), dim3((a.T * a.S + kWaves - 1) / kWaves), dim3(kThreads), 0, s, a);
    if (a.verdict) {
        if (!a.decides) hipLaunchKernelGGL((kq_verify_decide_kernel<DT>), dim3(a.B), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL((kq_verify_rest_kernel<DT, PT>), dim3((a.S + kWaves - 1) / kWaves, a.B), dim3(kThreads), 0, s, a);
    }
    hipLaunchKernelGGL((kq_verify_pick_kernel<DT, PT>), dim3(a.B), dim3(kThreads), 0, s, a);
}

template <int DT>
void launch_probs(const VerifyArgs &a, hipStream_t s) {
    if (!a.probs || a.probs_type == KQ_DTYPE_F32) launch<DT, KQ_DTYPE_F32>(a, s);
    else if (a.probs_type == KQ_DTYPE_BF16) launch<DT, KQ_DTYPE_BF16>(a, s);
    else launch<DT, KQ_DTYPE_F16>(a, s);
}

bool a_type(int dtype) { return dtype == KQ_DTYPE_F32 || dtype == KQ_DTYPE_F16 || dtype == KQ_DTYPE_BF16; }

}  // namespace

extern "C" {

size_t kq_verify_workspace_bytes(int32_t T, int32_t B, int32_t V, int dtype, int with_probs) {
    if (T < 1 || B < 1 || V < 1 || !a_type(dtype)) return 0;
    const int S = slices(V, dtype);
    return sizes_fit(T, B, V, S) ? need_bytes(T, B, S, with_probs != 0) : 0;
}

int kq_verify_drafts(const void *logits, int dtype, int64_t row_stride, const int32_t *tokens, const int32_t *cu_rows,
                     const float *uniforms, const float *draws, const void *draft_probs, int probs_dtype,
                     int64_t probs_row_stride, const float *temperatures, double temperature, const int32_t *kv_lens,
                     int32_t T, int32_t B, int32_t V, int32_t *accepted, int32_t *next_tokens, int32_t *keep_lens,
                     void *workspace, size_t workspace_bytes, kq_stream_t stream) {
    if (B == 0) return KQ_OK;
    const bool greedy_all = !temperatures && temperature == 0.0;
    if (!cu_rows || !accepted || !next_tokens || (keep_lens && !kv_lens) || (T > 0 && (!logits || !tokens)) ||
        (!greedy_all && ((T > 0 && !uniforms) || !draws)))
        return KQ_ERR_NULL_POINTER;
    if (!a_type(dtype) || (draft_probs && !a_type(probs_dtype))) return KQ_ERR_UNSUPPORTED_DTYPE;
    if (T < 0 || B < 0 || V < 1 || row_stride < 0 || (draft_probs && probs_row_stride < 0)) return KQ_ERR_BAD_SHAPE;
    if (!temperatures && !(temperature >= 0.0 && temperature <= 1.7976931348623157e308)) return KQ_ERR_BAD_ARGUMENT;
    if (((uintptr_t)logits & (dtype == KQ_DTYPE_F32 ? 3 : 1)) ||
        (draft_probs && ((uintptr_t)draft_probs & (probs_dtype == KQ_DTYPE_F32 ? 3 : 1))))
        return KQ_ERR_BAD_ALIGN;
    const int S = slices(V, dtype);
    if (!sizes_fit(T, B, V, S)) return KQ_ERR_BAD_SHAPE;
    if (T && (!workspace || workspace_bytes < need_bytes(T, B, S, draft_probs != nullptr))) return KQ_ERR_WORKSPACE_TOO_SMALL;
    if ((uintptr_t)workspace & 255) return KQ_ERR_BAD_ALIGN;
    VerifyArgs a;
    a.logits = logits;
    a.probs = draft_probs;
    a.stride = row_stride;
    a.probs_stride = probs_row_stride;
    a.tokens = tokens;
    a.cu = cu_rows;
    a.kv = kv_lens;
    a.u = uniforms;
    a.draws = draws;
    a.temps = temperatures;
    // (at either limit fp32 logits are as far apart, or as near, as past it, and the rate is finite and not 0)
    a.rate = temperature > 0.0 ? rate_at(std::min(std::max(temperature, 1e-300), 1e300)) : 0.0;
    a.T = T;
    a.B = B;
    a.V = V;
    a.S = S;
    a.probs_type = probs_dtype;
    a.part = (Part *)workspace;
    const bool with_rest = draft_probs && T && !greedy_all && S > kFewSlices;
    a.decides = (int64_t)B * ((S + kWaves - 1) / kWaves) <= kDecide;
    a.verdict = with_rest ? (Verdict *)((char *)workspace + part_bytes(T, S)) : nullptr;
    a.rest = with_rest ? (double *)(a.verdict + B) : nullptr;
    a.accepted = accepted;
    a.next = next_tokens;
    a.keep = keep_lens;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == KQ_DTYPE_F32) launch_probs<KQ_DTYPE_F32>(a, s);
    else if (dtype == KQ_DTYPE_BF16) launch_probs<KQ_DTYPE_BF16>(a, s);
    else launch_probs<KQ_DTYPE_F16>(a, s);
    return hipGetLastError() == hipSuccess ? KQ_OK : KQ_ERR_LAUNCH_FAILED;
}

}  // extern "C"
