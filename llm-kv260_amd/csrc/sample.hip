// The sampler's draw (include/w4a8_step.h; board/tp/tp_llama.cpp:894-936).
//
// Tokens are ordered by (logit descending, index ascending): the ascending
// order of comp = ~ordered(logit) << 32 | index. Every kept set is a prefix of
// that order, so top-k, top-p and the draw are one operation: the first token
// at which a running count or mass passes a target. No sort is needed for it.
//
// w = exp((l - max) / temperature) is taken in float64 and held as a multiple
// of 2^-44 in 64-bit integers: sums are exact, whatever their order. w below
// 2^-45 (31.2 nats under the largest) is 0 and such tokens are left out.
//
// Three launches over slices of the rows (one compute unit alone reads a row
// of 128256 logits in 30 us):
//   1. each slice's largest logit;
//   2. with the row's largest known, the slice's histogram of masses and counts
//      over BINS equal steps of (max - l) / temperature (LDS atomics), added to
//      the row's;
//   3. the row's histogram gives every target's bin; each slice lists its
//      tokens of those bins (some tens to hundreds: a bin is 1/33 nat), and the
//      row's last slice to be done narrows each bin down to its token.
// Narrowing: up to 64 tokens are compared with each other; more go into 1024
// finer steps of the wanted bins first, and only the target's step is compared;
// where even that holds more (ties), or the list overflows, histograms of comp
// over what is left of its range, 1024 steps at a time, read from the row if
// need be. A row of one slice does all of it in the third launch's workgroup,
// the only one then.
//
// Measured, 128256 logits: a row with top-k 40 16.1 us, with top-p 0.95 19.9, 64
// rows of all kinds 43.7 (0.75 TB/s); the launches of the first 2.9 + 5.3 + 9.2 in
// a profile, which adds a little to each, of the last 7.0 + 16.8 + 22.3. One pass over the
// bytes would take 0.1 and 6.9 us: few rows are bound by three launches that
// wait for each other and the third's prefix sums and list, many by the second's
// float64 exponentials and LDS atomics and the third's issue.
#include "../../include/w4a8_step.h"
#include "kernels.h"

namespace w4a8 {

namespace {

constexpr int BINS = 1024;
constexpr int ROW_THREADS = 512;       // the third launch's
constexpr int ALONE_THREADS = 1024;    // where it is the only one
constexpr int SLICE_THREADS = 512;
constexpr int SLICE = 4096;
constexpr int MAX_SLICES = 64;         // a lane each
constexpr int LIST = 4096;
constexpr int FEW = 64;                // tokens that are put in order by comparing all of them
constexpr uint64_t ONE = 1ull << 44;

__device__ __forceinline__ uint64_t comp_of(float l, int i) {
    const uint32_t b = __float_as_uint(l + 0.0f);              // -0 as +0
    const uint32_t ordered = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return (uint64_t)~ordered << 32 | (uint32_t)i;
}

__device__ __forceinline__ float logit_of(uint64_t comp) {
    const uint32_t ordered = ~(uint32_t)(comp >> 32);
    return __uint_as_float(ordered & 0x80000000u ? ordered ^ 0x80000000u : ~ordered);
}

// exp(x) 2^44 to the nearest integer for x in [-31.25, 0] (else: anything), off by less than 2^-48 of it before: exp(x)
// = 2^(i / 32) 2^k exp(r) with 32 k + i the integer nearest 32 x / ln 2 and |r| <= ln 2 / 64, the first factor from a
// table of 32 (LDS: a bank pair an entry), exp(r) by its series to r^5 (r^6 / 720 is 2^-48.7 at most). Sums with 3 2^51
// and 2^52 round to integers and leave them in the low bits; 2^k is added to the exponent's field.
constexpr int EXP_TABLE = 32;
__device__ __forceinline__ void exp_table_fill(double *table) {
    if (threadIdx.x < EXP_TABLE) table[threadIdx.x] = exp2((double)threadIdx.x / EXP_TABLE);
}
__device__ __forceinline__ uint64_t exp_units(double x, const double *table) {
    const double z = fma(x, EXP_TABLE * 1.4426950408889634074, 0x1.8p52);
    const int i = (int)(uint32_t)__double_as_longlong(z);
    const double r = fma(z - 0x1.8p52, -0.69314718055994530942 / EXP_TABLE, x);
    double e = fma(r, 1.0 / 120, 1.0 / 24);
    e = fma(r, e, 1.0 / 6);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    e *= table[i & (EXP_TABLE - 1)];
    e = __longlong_as_double(__double_as_longlong(e) + ((long long)((uint32_t)(44 + (i >> 5)) << 20) << 32));
    return (uint64_t)__double_as_longlong(e + 0x1p52) & 0xFFFFFFFFFFFFFull;
}

// A row's weights: what its settings and its largest logit make of a logit.
struct Weights {
    float top;
    double inv_t;
    float bin_scale;
    const double *table;
    // In units of 2^-44; 0 for what is never drawn (NaN and -inf among it).
    __device__ __forceinline__ uint64_t mass(float l) const {
        const double x = l == top ? 0.0 : ((double)l - (double)top) * inv_t;   // top = inf: -inf for the others
        const uint64_t m = exp_units(x, table);
        return x >= -31.25 ? m : 0;
    }
    // Never decreasing as l falls: every step of it is a rounded monotonic operation. The last bin starts 31.22 nats
    // down, past the last mass: it holds nothing that is drawn (but what is so far from the largest that the float32
    // difference is infinite, at temperatures as large).
    __device__ __forceinline__ float step(float l) const {
        return l == top ? 0.0f : fminf((top - l) * bin_scale, (float)(BINS - 1));
    }
    __device__ __forceinline__ int bin(float l) const { return (int)step(l); }
};

__device__ __forceinline__ Weights weights_of(const w4a8_sampling &set, int row, float top, const double *table) {
    const float t = set.temperature_rows ? set.temperature_rows[row] : set.temperature;
    Weights w;
    w.top = top;
    w.inv_t = t > 0.0f ? 1.0 / (double)t : 1.0;
    w.bin_scale = (float)(w.inv_t * (BINS / 31.25));
    w.table = table;
    return w;
}

__device__ __forceinline__ float min_p_of(const w4a8_sampling &set, int row) {
    return set.min_p_rows ? set.min_p_rows[row] : set.min_p;
}
__device__ __forceinline__ int top_k_of(const w4a8_sampling &set, int row) {
    return set.top_k_rows ? set.top_k_rows[row] : set.top_k;
}
// The least mass that min-p keeps; 0: all (min_p <= 0 or NaN).
__device__ __forceinline__ uint64_t least_mass(float min_p) {
    const double least = ceil((double)min_p * (double)ONE);
    return least > 0.0 ? (uint64_t)(least < 0x1p50 ? least : 0x1p50) : 0;
}

// The largest of a workgroup's values; red: a float a wave, free after the caller's next barrier.
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float *red) {
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v = fmaxf(v, red[i]);
    return v;
}

template <int THREADS>
__device__ __forceinline__ uint64_t block_sum(uint64_t v, unsigned long long *red) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) v += red[i];
    return v;
}

// The logits of [begin, end), U a thread at a time: the next U on their way while f(logit, index) takes these. The
// first U are loaded when it is made. Past the end: -inf, no token.
template <int THREADS, int U>
struct Logits {
    const float *logits;
    int begin, end;
    float v[U];
    __device__ __forceinline__ Logits(const float *logits, int begin, int end) : logits(logits), begin(begin), end(end) {
        load(begin + threadIdx.x);
    }
    __device__ __forceinline__ void load(int base) {
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = logits[min(base + j * THREADS, end - 1)];
    }
    // f takes U logits and the index of the first; the others' are THREADS apart.
    template <class F>
    __device__ __forceinline__ void batches(F f) {
        for (int base = begin + threadIdx.x; base < end; base += U * THREADS) {
            float now[U];
#pragma unroll
            for (int j = 0; j < U; ++j) now[j] = base + j * THREADS < end ? v[j] : -INFINITY;
            if (base + U * THREADS < end) load(base + U * THREADS);
            f(now, base);
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {
        batches([&](const float (&now)[U], int base) {
#pragma unroll
            for (int j = 0; j < U; ++j) f(now[j], base + j * THREADS);
        });
    }
};

// What a row's slices share; the first launch clears it.
struct RowState {
    unsigned long long mass[BINS], above;       // above: mass of what min-p keeps
    unsigned int count[BINS];                   // where a top-k needs it
    unsigned int listed, done;
    float top[MAX_SLICES];
    unsigned long long list[LIST];
};

struct SampleArgs {
    const float *logits, *u;
    int32_t *tokens;
    int64_t stride;
    int n, slices, slice;                       // slices of `slice` logits a row
    w4a8_sampling set;
    RowState *rows;                             // workspace
};

__global__ __launch_bounds__(SLICE_THREADS) void slice_max_kernel(SampleArgs a) {
    __shared__ float red[SLICE_THREADS / 64];
    const int row = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
    RowState &r = a.rows[row];
    for (int i = s * SLICE_THREADS + threadIdx.x; i < BINS; i += a.slices * SLICE_THREADS) r.mass[i] = 0, r.count[i] = 0;
    if (s == 0 && threadIdx.x == 0) r.above = 0, r.listed = 0, r.done = 0;
    float top = -INFINITY;
    Logits<SLICE_THREADS, 8>(a.logits + row * a.stride, s * a.slice, min((s + 1) * a.slice, a.n))
        .each([&](float l, int) { top = fmaxf(top, l); });       // a NaN leaves the other
    top = block_max<SLICE_THREADS>(top, red);
    if (threadIdx.x == 0) r.top[s] = top;
}

// In every lane.
__device__ __forceinline__ float row_top(const SampleArgs &a, const RowState &r) {
    const int lane = threadIdx.x & 63;
    float top = lane < a.slices ? r.top[lane] : -INFINITY;
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    return top;
}

// The histogram of the logits, and this thread's part of the mass that min-p keeps (0 where it keeps all). A batch's
// masses first, side by side: each alone is a chain of twenty float64 operations.
template <int THREADS, int U>
__device__ __forceinline__ uint64_t histogram(Logits<THREADS, U> &logits, const Weights &w, bool counts, float min_p,
                                              unsigned long long *mass, unsigned int *count) {
    const uint64_t least = least_mass(min_p);
    uint64_t above = 0;
    logits.batches([&](const float (&l)[U], int) {
        uint64_t m[U];
#pragma unroll
        for (int j = 0; j < U; ++j) m[j] = w.mass(l[j]);
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (m[j]) {
                const int b = w.bin(l[j]);
                atomicAdd(&mass[b], (unsigned long long)m[j]);
                if (counts) atomicAdd(&count[b], 1u);
            }
        if (least)
#pragma unroll
            for (int j = 0; j < U; ++j) above += m[j] >= least ? m[j] : 0;
    });
    return above;
}

__global__ __launch_bounds__(SLICE_THREADS) void slice_histogram_kernel(SampleArgs a) {
    __shared__ unsigned long long mass[BINS], red[SLICE_THREADS / 64];
    __shared__ unsigned int count[BINS];
    __shared__ double table[EXP_TABLE];
    const int row = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
    Logits<SLICE_THREADS, 8> logits(a.logits + row * a.stride, s * a.slice, min((s + 1) * a.slice, a.n));
    RowState &r = a.rows[row];
    exp_table_fill(table);
    for (int i = threadIdx.x; i < BINS; i += SLICE_THREADS) mass[i] = 0, count[i] = 0;
    const Weights w = weights_of(a.set, row, row_top(a, r), table);
    const bool counts = top_k_of(a.set, row) > 0;
    __syncthreads();
    uint64_t above = histogram(logits, w, counts, min_p_of(a.set, row), mass, count);
    above = block_sum<SLICE_THREADS>(above, red);   // its barrier: the histogram is whole
    if (threadIdx.x == 0) atomicAdd(&r.above, (unsigned long long)above);
    for (int i = threadIdx.x; i < BINS; i += SLICE_THREADS) {
        if (mass[i]) atomicAdd(&r.mass[i], mass[i]);
        if (counts && count[i]) atomicAdd(&r.count[i], count[i]);
    }
}

struct Shared {
    unsigned long long before_mass[BINS];      // of each bin, in the row
    unsigned int before_count[BINS];
    unsigned long long mass[BINS];             // histograms
    unsigned int count[BINS];
    unsigned long long list[LIST];
    unsigned long long wave_mass[16], low[16], high[16], before, left, answer_mass, answer;
    double table[EXP_TABLE];
    unsigned int wave_count[16], listed, base, few;
    int bin, last;
    float top[16];
    // A few tokens being compared, where no histogram is held.
    __device__ __forceinline__ unsigned long long *few_comp() { return mass; }
    __device__ __forceinline__ unsigned long long *few_mass() { return mass + FEW; }
    __device__ __forceinline__ unsigned int *few_bin() { return count; }
};

// BINS values of each kind over a workgroup, B = BINS / THREADS consecutive ones a thread.
template <int THREADS>
struct Bins {
    static constexpr int B = BINS / THREADS;
    uint64_t mass[B], mass_all;                // after scan(): what is before, and all
    uint32_t count[B], count_all;
    __device__ __forceinline__ int at(int j) const { return B * threadIdx.x + j; }
    __device__ __forceinline__ void load(const unsigned long long *m, const unsigned int *c) {
#pragma unroll
        for (int j = 0; j < B; ++j) mass[j] = m[at(j)], count[j] = c[at(j)];
    }
    __device__ __forceinline__ void store(unsigned long long *m, unsigned int *c) const {
#pragma unroll
        for (int j = 0; j < B; ++j) m[at(j)] = mass[j], c[at(j)] = count[j];
    }
    __device__ __forceinline__ void scan(Shared &s) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        uint64_t m = 0;
        uint32_t c = 0;
#pragma unroll
        for (int j = 0; j < B; ++j) m += mass[j], c += count[j];
        const uint64_t own_m = m;
        const uint32_t own_c = c;
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t pm = __shfl_up((unsigned long long)m, d);
            const uint32_t pc = __shfl_up(c, d);
            if (lane >= d) m += pm, c += pc;
        }
        if (lane == 63) s.wave_mass[wave] = m, s.wave_count[wave] = c;
        __syncthreads();
        m -= own_m;
        c -= own_c;
        mass_all = 0;
        count_all = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) {
            if (i < wave) m += s.wave_mass[i], c += s.wave_count[i];
            mass_all += s.wave_mass[i];
            count_all += s.wave_count[i];
        }
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const uint64_t here = mass[j];
            const uint32_t n = count[j];
            mass[j] = m;
            count[j] = c;
            m += here;
            c += n;
        }
    }
};

struct Found {
    uint64_t comp;     // the token
    uint64_t mass;     // the running mass, the token's included
};

// Within bin `bin`, the token at which the running mass (by_mass) or count passes `left`; `before`: the mass of the
// bins before. The bin's tokens are looked for in the list, or (a list that overflowed) in the row.
template <int THREADS>
__device__ __forceinline__ Found narrow(const Weights &w, int bin, bool by_mass, uint64_t left, uint64_t before,
                                        Shared &s, const float *row, int n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool in_row = s.listed > LIST;
    if (!in_row) n = (int)s.listed;
    uint64_t lo = 0, hi = ~0ull;
    const auto each = [&](auto f) {
        for (int base = tid; base < n; base += 4 * THREADS) {
            uint64_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = min(base + j * THREADS, n - 1);
                c[j] = in_row ? comp_of(row[i], i) : s.list[i];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (base + j * THREADS < n && c[j] >= lo && c[j] <= hi && w.bin(logit_of(c[j])) == bin) {
                    const uint64_t m = w.mass(logit_of(c[j]));
                    if (m) f(c[j], m);
                }
        }
    };
    for (int round = 0; round < 8; ++round) {       // 51 bits by ten a round: six, and the last look
        uint64_t low = ~0ull, high = 0;
        each([&](uint64_t c, uint64_t) { low = min(low, c), high = max(high, c); });
        for (int d = 32; d; d >>= 1) {
            low = min(low, (uint64_t)__shfl_xor((unsigned long long)low, d));
            high = max(high, (uint64_t)__shfl_xor((unsigned long long)high, d));
        }
        __syncthreads();                            // the round's scratch is free
        if (lane == 0) s.low[wave] = low, s.high[wave] = high;
        for (int i = tid; i < BINS; i += THREADS) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        low = s.low[0], high = s.high[0];
        for (int i = 1; i < THREADS / 64; ++i) low = min(low, (uint64_t)s.low[i]), high = max(high, (uint64_t)s.high[i]);
        if (low >= high) return Found{low, before + w.mass(logit_of(low))};
        const int shift = max(0, 54 - __clzll((long long)(high - low)));
        each([&](uint64_t c, uint64_t m) {
            atomicAdd(&s.mass[(c - low) >> shift], (unsigned long long)m);
            if (!by_mass) atomicAdd(&s.count[(c - low) >> shift], 1u);
        });
        __syncthreads();
        Bins<THREADS> h, at;
        h.load(s.mass, s.count);
        at = h;
        at.scan(s);
#pragma unroll
        for (int j = 0; j < h.B; ++j) {
            const uint64_t pre = by_mass ? at.mass[j] : at.count[j], here = by_mass ? h.mass[j] : h.count[j];
            if (pre <= left && left < pre + here) {
                s.bin = h.at(j);
                s.before = at.mass[j];
                s.left = left - pre;
            }
        }
        __syncthreads();
        lo = low + ((uint64_t)s.bin << shift);
        hi = lo + ((1ull << shift) - 1);
        before += s.before;
        left = s.left;
    }
    return Found{lo, before};
}

// ALONE: a whole row a workgroup, of ALONE_THREADS. Else a slice, with half the threads: the steps of the bins' sums and
// of a token's search are the same few instructions in every wave, so fewer waves have less to issue (sixteen took 4300
// cycles to scan the bins; one row, top-k 40, 18.3 us with 1024 threads, 16.2 with 512, 16.3 with 256; 64 rows 56, 47
// and 52).
template <bool ALONE>
__global__ __launch_bounds__(ALONE ? ALONE_THREADS : ROW_THREADS) void row_kernel(SampleArgs a) {
    constexpr int THREADS = ALONE ? ALONE_THREADS : ROW_THREADS;
    constexpr int U = ALONE ? 4 : 8;
    __shared__ Shared s;
    const int row = ALONE ? blockIdx.x : blockIdx.x / a.slices, slice = ALONE ? 0 : blockIdx.x % a.slices;
    const int tid = threadIdx.x;
    const float *logits = a.logits + row * a.stride;
    // Everything that waits for nothing is asked for first: the slice's logits, the settings, the row's histogram.
    const int begin = ALONE ? 0 : slice * a.slice, end = ALONE ? a.n : min(begin + a.slice, a.n);
    Logits<THREADS, U> tokens(logits, begin, end);
    const float t = a.set.temperature_rows ? a.set.temperature_rows[row] : a.set.temperature;
    const float p = a.set.top_p_rows ? a.set.top_p_rows[row] : a.set.top_p;
    const int k = top_k_of(a.set, row);
    const float u = a.u[row];
    const bool greedy = !(t > 0.0f);
    Bins<THREADS> pre;
    uint64_t above = 0;
    float top;
    if constexpr (!ALONE) {
        const RowState &r = a.rows[row];
        pre.load(r.mass, r.count);
        above = r.above;
        top = row_top(a, r);
    } else {
        top = -INFINITY;
        Logits<THREADS, 8>(logits, 0, a.n).each([&](float l, int) { top = fmaxf(top, l); });
        top = block_max<THREADS>(top, s.top);
    }
    exp_table_fill(s.table);                                     // read past barriers only
    if (!(top > -INFINITY)) {
        if (slice == 0 && tid == 0) a.tokens[row] = -1;
        return;
    }
    const Weights w = weights_of(a.set, row, top, s.table);
    if constexpr (ALONE) {
        for (int i = tid; i < BINS; i += THREADS) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        Logits<THREADS, 2> all(logits, 0, a.n);
        above = histogram(all, w, k > 0, min_p_of(a.set, row), s.mass, s.count);
        above = block_sum<THREADS>(above, s.low);
        pre.load(s.mass, s.count);
    }
    pre.scan(s);
    pre.store(s.before_mass, s.before_count);
    const uint64_t mass_all = pre.mass_all;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    // The last bin with no more than `target` before it, which is the one that the target falls in: every wave for
    // itself, over each sixty-fourth of them and then the sixty-four that follow.
    const auto find = [&](const auto *before, auto target) {
        const int lane = tid & 63;
        const int c = __popcll(__builtin_amdgcn_ballot_w64(before[64 * (lane & 15)] <= target) & 0xFFFF) - 1;
        return 64 * c + __popcll(__builtin_amdgcn_ballot_w64(before[64 * c + lane] <= target)) - 1;
    };
    const auto until = [&](int bin) { return bin + 1 < BINS ? (uint64_t)s.before_mass[bin + 1] : mass_all; };
    const auto at_least_one = [](uint64_t m) { return m > ONE ? m : ONE; };   // the first token is always kept
    const auto top_p_target = [&](uint64_t total) {
        const double need = ceil((double)p * (double)total);
        return need > 1.0 ? min((uint64_t)need, total) - 1 : 0;
    };
    const auto draw_target = [&](uint64_t total) {
        const double at = u > 0.0f && !greedy ? (double)u * (double)total : 0.0;
        return at < (double)total ? min((uint64_t)at, total - 1) : total - 1;
    };
    const bool by_min_p = least_mass(min_p_of(a.set, row)) != 0;
    const auto within_min_p = [&](uint64_t total) { return by_min_p ? at_least_one(min(total, above)) : total; };

    // The bins of the k-th token, of top-p's last and of the draw: each target is known up to the mass of the bin
    // that the one before falls in, so they are ranges, a bin or a few wide.
    const bool by_k = !greedy && k > 0 && (uint32_t)k < pre.count_all, by_p = !greedy && p < 1.0f;
    uint64_t least = mass_all, most = mass_all;
    int k_bin = -1, p_first = 0, p_last = -1;
    if (by_k) {
        k_bin = find(s.before_count, (unsigned int)k - 1);
        least = at_least_one(s.before_mass[k_bin]);
        most = until(k_bin);
    }
    if (by_p) {
        p_first = find(s.before_mass, top_p_target(least));
        p_last = find(s.before_mass, top_p_target(most));
        least = at_least_one(s.before_mass[p_first]);
        most = min(most, until(p_last));
    }
    if (greedy) least = most = ONE;
    const int d_first = find(s.before_mass, draw_target(within_min_p(least)));
    const int d_last = find(s.before_mass, draw_target(within_min_p(most)));

    // Their tokens.
    const auto wanted = [&](int b) {
        return b == k_bin || (b >= p_first && b <= p_last) || (b >= d_first && b <= d_last);
    };
    const float past = (float)(max(max(k_bin, p_last), d_last) + 1);
    tokens.batches([&](const float (&l)[U], int i) {
        // One place taken in the list a wave and batch, the lanes' own by counting.
        uint64_t hits[U];
        unsigned int all = 0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const float at = w.step(l[j]);                       // mostly past them; a NaN is in the last bin
            hits[j] = __builtin_amdgcn_ballot_w64(at < past && wanted((int)at) && l[j] > -INFINITY);
            all += (unsigned int)__popcll(hits[j]);
        }
        if (all == 0) return;
        unsigned int to = 0;
        if ((tid & 63) == 0) to = atomicAdd(&s.listed, all);
        to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const unsigned int at = to + __builtin_amdgcn_mbcnt_hi((unsigned int)(hits[j] >> 32),
                                                                   __builtin_amdgcn_mbcnt_lo((unsigned int)hits[j], 0));
            if ((hits[j] >> (tid & 63) & 1) && at < LIST) s.list[at] = comp_of(l[j], i + j * THREADS);
            to += (unsigned int)__popcll(hits[j]);
        }
    });
    __syncthreads();
    if constexpr (!ALONE) {
        // Into the row's list; the last slice to have done so reads it back. The entries are written through to the
        // device's coherence point and waited for before the barrier in front of the ticket, and read from there: no
        // cache is written back or dropped for them (a release and acquire a slice took 50 us of 64 rows' 174).
        RowState &r = a.rows[row];
        const unsigned int mine = s.listed;
        if (mine) {
            if (tid == 0) s.base = atomicAdd(&r.listed, mine);
            __syncthreads();
            for (unsigned int i = tid; i < mine && s.base + i < LIST && i < LIST; i += THREADS)
                __hip_atomic_store(&r.list[s.base + i], s.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (tid == 0)
            s.last = __hip_atomic_fetch_add(&r.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                     (unsigned int)a.slices - 1;
        __syncthreads();
        if (!s.last) return;
        const unsigned int listed = __hip_atomic_load(&r.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (unsigned int i = tid; i < listed && i < LIST; i += THREADS)
            s.list[i] = __hip_atomic_load(&r.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0) s.listed = listed;
        __syncthreads();
    }

    const int listed = (int)s.listed;
    if (listed <= FEW) {
        // Each token's running mass m and rank c: its bin's, and its bin's tokens before it, looked for by a group of
        // threads a token.
        if (tid < listed) {
            const float l = logit_of(s.list[tid]);
            s.few_mass()[tid] = w.mass(l);
            s.few_bin()[tid] = w.bin(l);
        }
        __syncthreads();
        constexpr int group = THREADS / FEW;
        const int i = tid / group, me = min(i, listed - 1);
        const uint64_t comp = s.list[me], mine = s.few_mass()[me];
        const unsigned int bin = s.few_bin()[me];
        uint64_t m = 0;
        uint32_t c = 0;
        for (int j = tid % group; j < listed; j += group)
            if (s.few_bin()[j] == bin && s.list[j] < comp) m += s.few_mass()[j], ++c;
        for (int d = 1; d < group; d <<= 1) {
            m += __shfl_xor((unsigned long long)m, d);
            c += __shfl_xor(c, d);
        }
        m += s.before_mass[bin];
        c += s.before_count[bin];
        const bool holds = i < listed && tid % group == 0 && mine != 0;
        uint64_t total = greedy ? ONE : mass_all;
        if (by_k) {
            if (holds && c == (uint32_t)k - 1) s.before = m + mine;
            __syncthreads();
            total = s.before;
        }
        if (by_p) {
            const uint64_t target = top_p_target(total);
            if (holds && m <= target && target < m + mine) s.left = m + mine;
            __syncthreads();
            total = s.left;
        }
        const uint64_t target = draw_target(within_min_p(total));
        if (holds && m <= target && target < m + mine) a.tokens[row] = (int32_t)(uint32_t)comp;
        return;
    }

    // More of them: a histogram of the wanted bins, each in as many steps as BINS slots give. slot_first, slot_rank:
    // the row's mass and count before a slot.
    // The wanted bins stand one after the other, each by the first of the three that it is wanted for: k's, top-p's, the
    // draw's.
    const int p_at = k_bin >= 0 ? 1 : 0, d_at = p_at + (p_last - p_first + 1), bins = d_at + (d_last - d_first + 1);
    const bool slots = listed <= LIST && bins <= BINS;
    const int per_bin = slots ? BINS >> (bins <= 1 ? 0 : 32 - __clz(bins - 1)) : 1;
    const auto slot_of = [&](float l) {
        const float at = w.step(l);
        const int b = (int)at;
        const int of = b == k_bin ? 0 : b >= p_first && b <= p_last ? p_at + b - p_first : d_at + b - d_first;
        return of * per_bin + (int)((at - (float)b) * (float)per_bin);
    };
    Bins<THREADS> slot, slot_first;
    if (slots) {
        for (int i = tid; i < BINS; i += THREADS) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        for (int i = tid; i < listed; i += THREADS) {
            const float l = logit_of(s.list[i]);
            const uint64_t m = w.mass(l);
            if (m == 0) continue;
            const int at = slot_of(l);
            atomicAdd(&s.mass[at], (unsigned long long)m);
            if (by_k) atomicAdd(&s.count[at], 1u);
        }
        __syncthreads();
        slot.load(s.mass, s.count);
        slot_first = slot;
        slot_first.scan(s);
        __syncthreads();
        slot_first.store(s.mass, s.count);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < slot.B; ++j) {
            const int of = slot.at(j) / per_bin;
            if (of >= bins) continue;                            // nothing in it
            const int b = of < p_at ? k_bin : of < d_at ? p_first + of - p_at : d_first + of - d_at;
            slot_first.mass[j] += s.before_mass[b] - s.mass[of * per_bin];
            slot_first.count[j] += s.before_count[b] - s.count[of * per_bin];
        }
    }

    // The k-th token, top-p's last and the draw, each from the mass that the one before leaves.
    uint64_t total = greedy ? ONE : mass_all;
    for (int stage = by_k ? 0 : by_p ? 1 : 2;; stage = stage == 0 && by_p ? 1 : 2) {
        const uint64_t target = stage == 0   ? (uint64_t)k - 1
                                : stage == 1 ? top_p_target(total)
                                             : draw_target(within_min_p(total));
        Found f{};
        unsigned int few = FEW + 1;
        if (slots) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < slot.B; ++j) {
                const uint64_t first = stage == 0 ? slot_first.count[j] : slot_first.mass[j];
                const uint64_t here = stage == 0 ? slot.count[j] : slot.mass[j];
                if (first <= target && target < first + here) {
                    s.bin = slot.at(j);
                    s.before = slot_first.mass[j];
                    s.left = target - first;
                }
            }
            if (tid == 0) s.few = 0;
            __syncthreads();
            for (int i = tid; i < listed; i += THREADS) {
                const float l = logit_of(s.list[i]);
                if (slot_of(l) != s.bin) continue;
                const uint64_t m = w.mass(l);
                if (m == 0) continue;
                const unsigned int at = atomicAdd(&s.few, 1u);
                if (at < FEW) s.few_mass()[at] = m, s.few_comp()[at] = s.list[i];
            }
            __syncthreads();
            few = s.few;
            if (few <= FEW) {
                if (tid < (int)few) {
                    const uint64_t comp = s.few_comp()[tid];
                    uint64_t m = 0, c = 0;
                    for (unsigned int j = 0; j < few; ++j)
                        if (s.few_comp()[j] < comp) m += s.few_mass()[j], ++c;
                    if (stage == 0 ? c == s.left : m <= s.left && s.left < m + s.few_mass()[tid]) {
                        s.answer = comp;
                        s.answer_mass = s.before + m + s.few_mass()[tid];
                    }
                }
                __syncthreads();
                f = Found{s.answer, s.answer_mass};
            }
        }
        if (few > FEW) {
            const int bin = stage == 0 ? find(s.before_count, (unsigned int)target) : find(s.before_mass, target);
            const uint64_t before = s.before_mass[bin];
            f = narrow<THREADS>(w, bin, stage != 0, target - (stage == 0 ? s.before_count[bin] : before), before, s,
                                logits, a.n);
        }
        total = f.mass;
        if (stage == 2) {
            if (tid == 0) a.tokens[row] = (int32_t)(uint32_t)f.comp;
            return;
        }
    }
}

// Slices a row: of SLICE logits while that makes at most 64 of them and 512 workgroups, two a compute unit in the
// third launch (one row of 128256, top-k 40: 16.2 us with slices of 4096, 16.8 of 2048 with more workgroups; 64 rows
// 47 and 49).
// One, the whole row a workgroup in one launch, past 170 rows, where two would be left (180 rows of 32000, top-k 40:
// 28.9 us whole, 35.9 in two; of 64000 46.9 and 54.7), and where it is done before the three launches of the slices:
// a workgroup takes n logits in the time in which all take 200 n, plus what the launches cost, that of some 1.9
// million (one row of 9000 15.3 whole and 16.1 sliced, 17.8 and 15.9 of 16000; 90 rows of 16000 18.9 and 21.7, 64 of
// 32000 27.0 and 23.5, 128 of 32000 27.8 and 28.2). Past 170 rows the rule looks at neither the vocabulary nor the CUs: a
// workgroup fills one, so up to 256 rows of 128256 are faster whole (256: 110 and 123 in three), 300 are not (177 whole,
// 154 in two, 142 in three), 512 are again (207 and 220).
int sample_slices(int m, int n) {
    if (m > 170 || (int64_t)n * (200 - m) <= 1900000) return 1;
    const int most = 512 / m < MAX_SLICES ? 512 / m : MAX_SLICES;
    const int s = (n + SLICE - 1) / SLICE;
    return s < most ? s : most;
}

}  // namespace

size_t sample_workspace_bytes(int m, int n) {
    return sample_slices(m, n) > 1 ? (size_t)m * sizeof(RowState) : 0;
}

hipError_t launch_sample(const float *logits, int64_t stride, int m, int n, const float *u, const w4a8_sampling &set,
                         int32_t *tokens, void *workspace, hipStream_t stream) {
    SampleArgs a{};
    a.logits = logits;
    a.u = u;
    a.tokens = tokens;
    a.stride = stride;
    a.n = n;
    a.set = set;
    a.slices = sample_slices(m, n);
    if (a.slices == 1) {
        hipLaunchKernelGGL(row_kernel<true>, dim3((unsigned)m), dim3(ALONE_THREADS), 0, stream, a);
        return hipGetLastError();
    }
    a.slice = (n + a.slices - 1) / a.slices;
    a.rows = static_cast<RowState *>(workspace);
    const unsigned all = (unsigned)(m * a.slices);
    hipLaunchKernelGGL(slice_max_kernel, dim3(all), dim3(SLICE_THREADS), 0, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(slice_histogram_kernel, dim3(all), dim3(SLICE_THREADS), 0, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(row_kernel<false>, dim3(all), dim3(ROW_THREADS), 0, stream, a);
    return hipGetLastError();
}

}  // namespace w4a8
