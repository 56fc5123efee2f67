// Attention of one new token a row over the paged cache (include/w4a8_step.h).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp2(s_j - ref),  s_j = (scale log2 e) q . k_j
//
// for any ref (a running maximum keeps p in range). K and V are read once:
// 4 len head_dim bytes a row and KV head against 4 G len head_dim operations
// for the G query heads that share them, so the memory is the bound, and the
// kernel is built to keep loads in flight:
//
//  * A wave takes 32 positions at a time, its next tile's K and V on their way
//    into registers while it computes: 64 D bytes a tile in plain 16-byte
//    loads of whole rows, no LDS, no barrier in the loop.
//  * Both products are 16x16x32 MFMAs with the heads as the N dimension
//    (up to 16; G = 1 wastes 15 columns, the matrix cores have room for it):
//    S^T = K Q^T takes K's rows as they are loaded. Its result leaves a lane
//    with eight positions of one head -- in the order in which P^T is the B
//    operand of O^T = V^T P^T, so P never crosses lanes; V^T's operand wants
//    eight positions of one dimension a lane, which a lane that loaded D / 16
//    dimensions of eight positions has: one v_perm a register.
//  * The cache's values are exact in the products, q and p are float32: each is
//    split into 16-bit parts whose sum holds 22 bits (fp16: 2 parts) or 24
//    (bf16: 3), one MFMA a part. fp16's exponents end 30 powers of two under a
//    head's largest |q|, and what lies 17 under it has fewer bits; p keeps its
//    bits at any size (Half).
//  * ref moves only when a score passes it by some powers of two (Half::LAZY; a
//    vote; about once in a row), so the loop has no exchange between lanes and no
//    rescaling.
//  * A row's positions are split over workgroups where rows and heads alone do
//    not fill the GPU, and the parts joined by a second launch.
//
// Measured, 32 heads over 8: two rows of 131072 (D 64, fp16) 88 us, 6.1 TB/s; 64
// rows of up to 8192 (D 128, bf16, ragged) 196 us, 5.8 TB/s; a row of 8192 (D 64,
// fp16) 9.6 us; a row of 300 (D 64, fp16) 6.0 us, of which the memory's share is
// under one: the launch, three dependent loads (table, K, V) and the waves' join.
#include "../../include/w4a8_step.h"
#include "kernels.h"
#include "kv_device.h"

namespace w4a8 {

namespace {

constexpr int TILE = 32;          // positions a wave takes at a time
constexpr int WAVES = 4;
constexpr int HEADS = 16;         // columns: query heads a workgroup takes, of a row or of several
constexpr int MAX_SPLITS = 256;   // of a row: the join gives each a thread

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Half;
template <>
struct Half<f16_t> {
    using vec = f16x8;
    static constexpr int PARTS = 2;
    static constexpr uint32_t EXPONENT = 0x7C00;
    static constexpr bool SCALED = true;    // q is brought to fp16's range by a power of two a head
    static constexpr float LAZY = 4.0f;     // scores may pass ref by it before ref moves
    // log2 of what stands for a p of 1 at ref: p is at most 2^15, half of fp16's range.
    static __device__ __forceinline__ float unit(int) { return 15.0f - LAZY; }
    // p's parts: its rounding to fp16, and 2^12 times what that leaves (2^3 at most), whose products are scaled back in
    // float32. Together they hold 22 bits down to fp16's least normal, 2^-14, which is 2^-25 of a p at ref: a band. What
    // is under it is taken 2^29 times as large in a band of its own, and so on to float32's least. (An unscaled low part
    // would lose bits from 2^-10 of the largest p on, and hold nothing under 2^-32.) The scale costs D / 4 multiply-adds a
    // lane and tile and the wait for the low products: one to three percent (two rows of 131072 of D 64 87.6 -> 88.6 us, 24
    // of 640 15.4 -> 15.6), a row of 300 5.5 -> 5.9; rows whose scores all lie 17 nats apart, a second band in every tile,
    // 97 us of the 87.6.
    static constexpr float LOW = 0x1p12f, LEAST = 0x1p-14f, BAND = 0x1p29f;
    static __device__ __forceinline__ f32x4 mfma(vec a, vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<bf16_t> {
    using vec = bf16x8;
    static constexpr int PARTS = 3;
    static constexpr uint32_t EXPONENT = 0x7F80;
    static constexpr bool SCALED = false;
    static constexpr float LAZY = 8.0f;
    // V may be as large as a float32: p is at most 1 / len, so that no sum of p v passes the largest v. What is left of
    // float32's range below holds p to 22 bits down to 2^-64 of the row's largest, and none under 2^-88 (len = 2^30).
    static __device__ __forceinline__ float unit(int len) {
        return -LAZY - (float)(len > 1 ? 32 - __builtin_clz((unsigned)(len - 1)) : 0);
    }
    static __device__ __forceinline__ f32x4 mfma(vec a, vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// x as PARTS 16-bit values that add up to it, each the rounding of what the ones before leave.
template <class T>
__device__ __forceinline__ void split8(const float (&x)[8], typename Half<T>::vec (&out)[Half<T>::PARTS]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
    for (int p = 0; p < Half<T>::PARTS; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            out[p][j] = (T)rest[j];
            rest[j] -= (float)out[p][j];
        }
}

// fp16's two parts of p, the second scaled (Half::LOW).
template <class T>
__device__ __forceinline__ void split_scaled(const float (&p)[8], typename Half<T>::vec (&out)[2]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        out[0][j] = (T)p[j];
        out[1][j] = (T)((p[j] - (float)out[0][j]) * Half<T>::LOW);
    }
}

// Whether any lane's p has values under its band (Half::LEAST; 0 is none, NaN stays in p): if so they go from p to
// `under`, scaled to the next.
template <class T>
__device__ __forceinline__ bool next_band(float (&p)[8], float (&under)[8]) {
    uint32_t least = ~0u;               // of the bits less one: 0 comes last
#pragma unroll
    for (int j = 0; j < 8; ++j) least = min(least, __float_as_uint(p[j]) - 1);
    if (__builtin_amdgcn_ballot_w64(least < __float_as_uint(Half<T>::LEAST) - 1) == 0) return false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool small = p[j] < Half<T>::LEAST;
        under[j] = small ? p[j] * Half<T>::BAND : 0.0f;
        p[j] = small ? 0.0f : p[j];
    }
    return true;
}

struct AttendArgs {
    const float *q;
    const void *k, *v;
    const int32_t *table, *pos;
    float *out, *part, *part_ml;
    int64_t table_stride;
    int m, rows_each;                   // rows, and how many of them a workgroup takes (one but with SHARED)
    int heads, group, head_tiles;       // query heads, of one KV head, tiles of HEADS of those
    int kv_heads, pages, page_shift, table_pages;
    int splits;
    float scale;                        // times log2 e
};

// How K and V are read: through the caches; past them; or once for several rows of one table (a prompt's tokens), whose
// heads fill the columns together.
enum Reading { CACHED, STREAMED, SHARED };

// A row's tiles go round its splits, WAVES at a time: split s takes the rounds s, s + splits, ... Which tile a
// wave takes first does not hang on the row's length, so its page is looked up beside that.
__device__ __forceinline__ int splits_used(int len, int splits) {
    const int rounds = (len + TILE * WAVES - 1) / (TILE * WAVES);
    return rounds < splits ? rounds : splits;
}

// A tile's pages, one for each half of 16 positions (pages hold 16 at least), and its K and V.
template <int D>
struct Tile {
    typedef uint32_t v_row __attribute__((ext_vector_type(D / 32 == 8 ? 4 : D / 32), aligned(4)));
    static constexpr int V_LOADS = D / 32 == 8 ? 2 : 1;
    int page[2];
    u32x4 k[2][D / 32];
    v_row v[8][V_LOADS];
};

struct Pages {
    int of[2];
};
__device__ __forceinline__ Pages tile_pages(const AttendArgs &a, const int32_t *table, int tile) {
    return Pages{{kv_page(table, (tile * TILE) >> a.page_shift, a.table_pages, a.pages),
                  kv_page(table, (tile * TILE + 16) >> a.page_shift, a.table_pages, a.pages)}};
}

// A 16-byte or narrower load, past the caches' replacement (NT) where what is read is read once.
template <bool NT, class V>
__device__ __forceinline__ V load_once(const char *p) {
    if constexpr (NT)
        return __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
    else
        return *reinterpret_cast<const V *>(p);
}

// The loads of a tile whose pages are known. An absent page's come from page 0 (memory that is there), for nothing.
template <int D, bool NT>
__device__ __forceinline__ void tile_load(const AttendArgs &a, int kvh, int tile, Pages pages, int lane, Tile<D> &t) {
    const int n = lane & 15, g = lane >> 4;
    t.page[0] = pages.of[0];
    t.page[1] = pages.of[1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int slot = (tile * TILE + 16 * h) & ((1 << a.page_shift) - 1);
        const size_t at = 2 * (kv_offset(t.page[h] < 0 ? 0 : t.page[h], a.kv_heads, kvh, a.page_shift, D) + (size_t)slot * D);
        const char *k = (const char *)a.k + at + (uint32_t)(2 * n * D + 16 * g);
        const char *v = (const char *)a.v + at + (uint32_t)(2 * 4 * g * D + 2 * n * (D / 16));
#pragma unroll
        for (int c = 0; c < D / 32; ++c) t.k[h][c] = load_once<NT, u32x4>(k + 64 * c);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < Tile<D>::V_LOADS; ++i)
                t.v[4 * h + r][i] = load_once<NT, typename Tile<D>::v_row>(v + 2 * r * D + 16 * i);
    }
}

// Q^T's operand: lane (g, n) takes dimensions 32 c + 8 g .. + 7 of head n, in
// PARTS parts. In registers, or, at D = 256 where those would be 96, in LDS:
// 24 reads of 16 bytes a tile at most, against the 32 KB that the tile is.
template <class T, int D>
struct Query {
    using H = Half<T>;
    static constexpr bool LDS = D > 128;
    using Store = typename H::vec[LDS ? D / 32 * H::PARTS * 64 : 1];
    typename H::vec reg[LDS ? 1 : D / 32][H::PARTS];
    typename H::vec *lds;
    int exp;                            // the power of two that the head's scores are to be scaled by
    __device__ __forceinline__ void put(int c, const typename H::vec (&v)[H::PARTS], int lane, int wave) {
#pragma unroll
        for (int p = 0; p < H::PARTS; ++p) {
            if constexpr (!LDS)
                reg[c][p] = v[p];
            else if (c % WAVES == wave)
                lds[(c * H::PARTS + p) * 64 + lane] = v[p];
        }
    }
    __device__ __forceinline__ typename H::vec get(int c, int p, int lane) const {
        if constexpr (LDS)
            return lds[(c * H::PARTS + p) * 64 + lane];
        else
            return reg[c][p];
    }
};

// Positions: the lane's column's own, and the least and most of the workgroup's; Half::unit of the most, which all splits
// of a row share.
struct Lens {
    int own, least, most;
    float unit;
};

template <class T, int D>
struct State {
    f32x4 o[D / 16];
    float ref, sum;                     // of the lane's head; sum over the lane's own positions
};

template <class T, int D, bool ROWS>
__device__ __forceinline__ void tile_attend(const Query<T, D> &q, Tile<D> &t, int first, Lens len, int lane,
                                            State<T, D> &st) {
    using H = Half<T>;
    const int g = lane >> 4;
    float s[8];
    f32x4 acc[2] = {};
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int p = 0; p < H::PARTS; ++p) {
            const typename H::vec qv = q.get(c, p, lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[h] = H::mfma(__builtin_bit_cast(typename H::vec, t.k[h][c]), qv, acc[h]);
            // The reads of all chunks at once would not fit the registers.
            if (Query<T, D>::LDS && p == H::PARTS - 1 && c % 2) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[4 * h + r] = H::SCALED ? __builtin_amdgcn_ldexpf(acc[h][r], q.exp) : acc[h][r];
            // An infinite K meets q's parts one by one, with either sign: whatever that gives, the output is NaN (it is so
            // for +inf and NaN), for -inf would drop the position.
            if (s[4 * h + r] == -INFINITY) s[4 * h + r] = NAN;
        }
    // Dimension n D / 16 + i of the lane's eight positions.
    uint32_t lows = 0x05040100u, highs = 0x07060302u;
    const auto operand = [&](int i) {
        const auto word = [&](int j) { return t.v[j][i / 8][(i % 8) / 2]; };
        const uint32_t sel = i & 1 ? highs : lows;
        return make_uint4(__builtin_amdgcn_perm(word(1), word(0), sel), __builtin_amdgcn_perm(word(3), word(2), sel),
                          __builtin_amdgcn_perm(word(5), word(4), sel), __builtin_amdgcn_perm(word(7), word(6), sel));
    };
    if (t.page[0] < 0 || t.page[1] < 0 || first + TILE > len.least) {
        // Masked positions: no score, and zeros for V where no row has stored any, whose bits may be anything.
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = first + 16 * h + 4 * g + r;
                if (t.page[h] < 0 || at >= len.own) s[4 * h + r] = -INFINITY;
                if (t.page[h] < 0 || at >= len.most)
#pragma unroll
                    for (int i = 0; i < Tile<D>::V_LOADS; ++i) t.v[4 * h + r][i] = 0;
            }
        // A position that one row attends and another does not holds the first one's V: where that is no number, its
        // product with the other's p of 0 is none either. It is taken out, and the outputs that it belongs to are none:
        // a product of its places with the columns that attend them tells which.
        if constexpr (ROWS) {
            // Bits 0 and 16: whether a word's halves are infinite or NaN, their exponents all ones.
            const auto odd = [&](uint32_t w) {
                constexpr uint32_t e = H::EXPONENT * 0x10001u, unit = (0x8000u - H::EXPONENT) * 0x10001u;
                return ((w & e) + unit) >> 15 & 0x10001u;
            };
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) any |= odd(t.v[j][i / 4][i % 4]);
            if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
                typename H::vec seen;
#pragma unroll
                for (int j = 0; j < 8; ++j) seen[j] = (T)(first + 16 * (j / 4) + 4 * g + j % 4 < len.own ? 1.0f : 0.0f);
                const uint32_t one = __builtin_bit_cast(uint16_t, (T)1.0f);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint4 v = operand(i);
                    const uint4 at = make_uint4(odd(v.x) * one, odd(v.y) * one, odd(v.z) * one, odd(v.w) * one);
                    const f32x4 some = H::mfma(__builtin_bit_cast(typename H::vec, at), seen, f32x4{});
#pragma unroll
                    for (int r = 0; r < 4; ++r) st.o[i][r] = some[r] > 0.0f ? NAN : st.o[i][r];
                    __builtin_amdgcn_sched_barrier(0);      // one at a time: this is rare, and its registers are not to be had
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) t.v[j][i / 4][i % 4] &= ~(odd(t.v[j][i / 4][i % 4]) * 0xFFFFu);
            }
        }
    }
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
    if (__builtin_amdgcn_ballot_w64(top > st.ref + H::LAZY) != 0) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float ref = fmaxf(st.ref, top);
        const float alpha = ref == st.ref ? 1.0f : __builtin_amdgcn_exp2f(st.ref - ref);
        st.ref = ref;
        st.sum *= alpha;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) st.o[i] *= alpha;
    }
    const float base = st.ref == -INFINITY ? 0.0f : st.ref - len.unit;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(s[j] - base);
    st.sum += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    typename H::vec p[H::PARTS];
    if constexpr (!H::SCALED) {
        split8<T>(s, p);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const auto v = __builtin_bit_cast(typename H::vec, operand(i));
#pragma unroll
            for (int b = 0; b < H::PARTS; ++b) st.o[i] = H::mfma(v, p[b], st.o[i]);
        }
    } else {
        const auto add_scaled = [](f32x4 x, float f, f32x4 &o) {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(x[r], f, o[r]);
        };
        float under[8], band = 1.0f;
        bool more = next_band<T>(s, under);
        split_scaled<T>(s, p);
        constexpr int AT_ONCE = D > 128 ? 2 : 4;         // low products on their way: registers
#pragma unroll
        for (int i = 0; i < D / 16; i += AT_ONCE) {
            f32x4 low[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE && i + j < D / 16; ++j) {
                const auto v = __builtin_bit_cast(typename H::vec, operand(i + j));
                low[j] = H::mfma(v, p[1], f32x4{});
                st.o[i + j] = H::mfma(v, p[0], st.o[i + j]);
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE && i + j < D / 16; ++j) add_scaled(low[j], 1.0f / H::LOW, st.o[i + j]);
        }
        // The bands under the first, one dimension tile after the other: few tiles have any.
        while (__builtin_expect(more, false)) {
            float now[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) now[j] = under[j];
            more = next_band<T>(now, under);
            split_scaled<T>(now, p);
            band *= 1.0f / H::BAND;
            // Other constants, as far as the compiler knows: it would keep all of V's operands from band to band. (Not
            // volatile, which would count as a store and make the page table's scalar loads vector ones.)
            __asm__("" : "+s"(lows), "+s"(highs));
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const auto v = __builtin_bit_cast(typename H::vec, operand(i));
                add_scaled(H::mfma(v, p[0], f32x4{}), band, st.o[i]);
                add_scaled(H::mfma(v, p[1], f32x4{}), band / H::LOW, st.o[i]);
            }
        }
    }
}

template <class T, int D, Reading READING>
__global__ __launch_bounds__(64 * WAVES, 2) void attend_kernel(AttendArgs a) {
    using H = Half<T>;
    constexpr bool NT = READING == STREAMED, ROWS = READING == SHARED;
    constexpr int PITCH = D + 4;         // LDS row of a head: rows start four banks apart
    constexpr int BATCH = D > 128 ? HEADS / 2 : HEADS;           // heads whose parts meet in LDS at a time
    __shared__ float refs[WAVES][HEADS], sums[WAVES][HEADS];
    __shared__ __attribute__((aligned(16))) float os[WAVES][BATCH * PITCH];
    __shared__ typename Query<T, D>::Store q_lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int b = blockIdx.x;
    const int split = b % a.splits;
    b /= a.splits;
    const int ht = b % a.head_tiles;
    b /= a.head_tiles;
    const int kvh = b % a.kv_heads, row = b / a.kv_heads * (ROWS ? a.rows_each : 1);
    const int32_t *table = a.table + row * a.table_stride;
    int tile = split * WAVES + wave;
    const int step = a.splits * WAVES;
    Pages pages = tile_pages(a, table, tile);
    const int n = lane & 15, g = lane >> 4;
    // Column c of this workgroup's is query head head_of(c) of all rows' (row, head) pairs; past the last: it again.
    const int here = ROWS ? min(a.rows_each, a.m - row) * a.group : min(a.group - ht * HEADS, HEADS);
    const auto head_of = [&](int c) {
        return ROWS ? (size_t)(row + c / a.group) * a.heads + kvh * a.group + c % a.group
                    : (size_t)row * a.heads + kvh * a.group + ht * HEADS + c;
    };
    const int column = min(n, here - 1);
    Lens len;
    if constexpr (ROWS) {
        len.own = kv_len(a.pos[row + column / a.group], a.table_pages, a.page_shift);
        int most = len.own, least = len.own;
        for (int d = 1; d < 16; d <<= 1) most = max(most, __shfl_xor(most, d)), least = min(least, __shfl_xor(least, d));
        len.most = __builtin_amdgcn_readfirstlane(most);
        len.least = __builtin_amdgcn_readfirstlane(least);
    } else {
        len.own = len.least = len.most = kv_len(a.pos[row], a.table_pages, a.page_shift);
    }
    len.unit = H::unit(len.most);
    const int used = splits_used(len.most, a.splits);
    if (split >= used && split > 0) return;
    const int end = (len.most + TILE - 1) / TILE;
    Tile<D> ta;

    // Every wave takes all of the heads' queries.
    Query<T, D> q;
    q.lds = q_lds;
    q.exp = 0;
    const float *src = a.q + head_of(column) * D + 8 * g;
    const auto scaled = [&](int c, float (&x)[8]) {
        const float4 u = *reinterpret_cast<const float4 *>(src + 32 * c), v = *reinterpret_cast<const float4 *>(src + 32 * c + 4);
        const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = f[j] * a.scale;
    };
    if constexpr (H::SCALED) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            float x[8];
            scaled(c, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        q.exp = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
    }
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        float x[8];
        scaled(c, x);
        if constexpr (H::SCALED)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_ldexpf(x[j], -q.exp);
        typename H::vec parts[H::PARTS];
        split8<T>(x, parts);
        q.put(c, parts, lane, wave);
    }
    if constexpr (Query<T, D>::LDS) __syncthreads();

    State<T, D> st;
    st.ref = -INFINITY;
    st.sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    if (tile < end) {
        tile_load<D, NT>(a, kvh, tile, pages, lane, ta);
        pages = tile_pages(a, table, tile + step);
        if constexpr (D > 128 || (ROWS && D > 96)) {
            // A tile is 128 registers (D = 128, rows of one table: 64): one at a time, two waves a SIMD or three to fill
            // each other's waits.
            for (;;) {
                tile_attend<T, D, ROWS>(q, ta, tile * TILE, len, lane, st);
                tile += step;
                if (tile >= end) break;
                tile_load<D, NT>(a, kvh, tile, pages, lane, ta);
                pages = tile_pages(a, table, tile + step);
            }
        } else {
            Tile<D> tb;
            for (;;) {
                const int next = tile + step;
                if (next < end) tile_load<D, NT>(a, kvh, next, pages, lane, tb);
                pages = tile_pages(a, table, next + step);
                tile_attend<T, D, ROWS>(q, ta, tile * TILE, len, lane, st);
                if (next >= end) break;
                tile = next + step;
                if (tile < end) tile_load<D, NT>(a, kvh, tile, pages, lane, ta);
                pages = tile_pages(a, table, tile + step);
                tile_attend<T, D, ROWS>(q, tb, next * TILE, len, lane, st);
                if (tile >= end) break;
            }
        }
    }

    // The waves' parts meet in LDS, brought to the largest of their refs.
    st.sum += __shfl_xor(st.sum, 16);
    st.sum += __shfl_xor(st.sum, 32);
    if (g == 0) refs[wave][n] = st.ref;
    __syncthreads();
    float ref = refs[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) ref = fmaxf(ref, refs[w][n]);
    const float mine = st.ref == ref ? 1.0f : __builtin_amdgcn_exp2f(st.ref - ref);
    if (g == 0) sums[wave][n] = st.sum * mine;
    const bool whole = used <= 1;
    for (int first = 0; first < here; first += BATCH) {
        __syncthreads();
        if (n >= first && n < min(first + BATCH, here)) {
#pragma unroll
            for (int r = 0; r < 4; ++r)      // lane (g, n): dimensions (4 g + r) D / 16 + i of head n
#pragma unroll
                for (int i = 0; i < D / 16; i += 2)
                    *reinterpret_cast<float2 *>(&os[wave][(n - first) * PITCH + (4 * g + r) * (D / 16) + i]) =
                        make_float2(st.o[i][r] * mine, st.o[i + 1][r] * mine);
        }
        __syncthreads();
        const int heads_now = min(BATCH, here - first);
        for (int e = threadIdx.x; e < heads_now * (D / 4); e += 64 * WAVES) {
            const int h = e / (D / 4), d = 4 * (e % (D / 4));
            float4 o = *reinterpret_cast<const float4 *>(&os[0][h * PITCH + d]);
            float sum = sums[0][first + h];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                const float4 p = *reinterpret_cast<const float4 *>(&os[w][h * PITCH + d]);
                o = make_float4(o.x + p.x, o.y + p.y, o.z + p.z, o.w + p.w);
                sum += sums[w][first + h];
            }
            const size_t head = head_of(first + h);
            if (whole) {
                o = sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                : make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum);
                *reinterpret_cast<float4 *>(a.out + head * D + d) = o;
            } else {
                *reinterpret_cast<float4 *>(a.part + (head * a.splits + split) * D + d) = o;
                if (d == 0) {
                    float m = refs[0][first + h];
                    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, refs[w][first + h]);
                    *reinterpret_cast<float2 *>(a.part_ml + 2 * (head * a.splits + split)) = make_float2(m, sum);
                }
            }
        }
    }
}

// A head's parts joined: out = sum_s 2^(ref_s - ref) o_s / sum_s 2^(ref_s - ref) sum_s. One workgroup a head, all of it
// latency: D / 4 threads take a part at a time, so 256 threads have 1024 / D parts on their way at once, four rounds
// of them before the first weight is known.
template <int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
    constexpr int COLS = D / 4, AT_ONCE = 256 / COLS, AHEAD = 4;
    __shared__ float weights[MAX_SPLITS], tops[4], totals[4];
    __shared__ float4 parts[AT_ONCE][COLS];
    const size_t head = blockIdx.x;
    const int row = blockIdx.x / a.heads, tid = threadIdx.x;
    const int col = tid % COLS, first = tid / COLS;      // D = 96: sixteen threads past the last slice idle
    // Parts past the row's own are loaded too (memory of the workspace, never used): no load waits for its length.
    const float4 *part = reinterpret_cast<const float4 *>(a.part + head * a.splits * D) + col;
    float4 v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (first < AT_ONCE && first + j * AT_ONCE < a.splits) v[j] = part[(size_t)(first + j * AT_ONCE) * COLS];
    float2 ml = tid < a.splits ? reinterpret_cast<const float2 *>(a.part_ml)[head * a.splits + tid] : make_float2(0.0f, 0.0f);
    // The length that its workgroups went by: the longest of the rows that they took together.
    int pos = a.pos[row];
    if (a.rows_each > 1)
        for (int i = row - row % a.rows_each, n = min(i + a.rows_each, a.m); i < n; ++i) pos = max(pos, a.pos[i]);
    const int used = splits_used(kv_len(pos, a.table_pages, a.page_shift), a.splits);
    if (used <= 1) return;
    if (tid >= used) ml = make_float2(-INFINITY, 0.0f);
    float ref = ml.x;
    for (int d = 32; d; d >>= 1) ref = fmaxf(ref, __shfl_xor(ref, d));
    if ((tid & 63) == 0) tops[tid >> 6] = ref;
    __syncthreads();
    ref = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float w = ml.x == ref ? 1.0f : __builtin_amdgcn_exp2f(ml.x - ref);
    if (tid < used) weights[tid] = w;
    float sum = tid < used ? w * ml.y : 0.0f;
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((tid & 63) == 0) totals[tid >> 6] = sum;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](float4 p, float f) {
        o = make_float4(fmaf(f, p.x, o.x), fmaf(f, p.y, o.y), fmaf(f, p.z, o.z), fmaf(f, p.w, o.w));
    };
    if (first < AT_ONCE) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (first + j * AT_ONCE < used) add(v[j], weights[first + j * AT_ONCE]);
        for (int s = first + AHEAD * AT_ONCE; s < used; s += AT_ONCE) add(part[(size_t)s * COLS], weights[s]);
        parts[first][col] = o;
    }
    __syncthreads();
    if (tid >= COLS) return;
    o = parts[0][tid];
#pragma unroll
    for (int s = 1; s < AT_ONCE; ++s) {
        const float4 p = parts[s][tid];
        o = make_float4(o.x + p.x, o.y + p.y, o.z + p.z, o.w + p.w);
    }
    sum = (totals[0] + totals[1]) + (totals[2] + totals[3]);
    reinterpret_cast<float4 *>(a.out + head * D)[tid] =
        sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum);
}

// Rows that a workgroup takes together: those of one table, as many as fill its columns. 32 heads over 8, fp16, in us,
// alone and together: a prompt of 16 rows (D 64) 4.1 and 4.8, 128 rows 7.4 and 5.1, 512 rows 36 and 14.6, 2048 rows 368
// and 104; D 128: 512 rows 57 and 20.5, 2048 rows 685 and 170. Bound by the reads from the caches, 10 TB/s at 2048 rows:
// every four rows read all of K and V. Rows drafted behind 32768 (D 64): two 26 and 18, eight 70 and 21; behind 2048 two
// 7.4 and 7.7, eight 10.4 and 8.2.
int attend_rows_each(int group, const w4a8_kv_rows &r) {
    return r.table_stride == 0 && r.m > 1 && group <= HEADS / 2 ? HEADS / group : 1;
}

// Splits of a row, by the length that its table allows (all that the host knows of it: a row of 300 takes 6.1 us with a
// table of its own width and 8.0 with one of 8192 or 131072, eight of up to 2048 14.1, 14.0 and 28.1) and what rows and
// heads leave of the GPU (groups of them; a round is the 128 positions that a workgroup's waves take at once). Measured,
// in us:
//  * up to three rounds, one: the join costs 2.5, a round 1 (300 positions, D 64, 6.1 against 7.2 in three splits; 512
//    positions, four rounds, D 128, 8.9 whole and 8.1 split; D 64 6.8 and 7.2).
//  * to eight rounds also where the groups alone give three quarters of the compute units one: no join, and the rows
//    need not be read in turn (24 rows of 640, 192 groups: 14.3 whole, 19.2 in three; 32 of 1024 at most, ragged: 20.0
//    and 23.9 in two; 16 of 1024, 128 groups: 20.2 and 17.8 in four).
//  * else to 512 workgroups, two a compute unit, a round each at least (one row of 8192: 9.9 with 64 splits, 10.9 with
//    16; sixteen of 2048: 31.7 with 512 workgroups, 32.4 with 1024, 36.6 with 2048; 128 rows of 1024: 98.5 whole,
//    109.6 in two).
//  * past that to 4096 while each has sixteen rounds: rows of unequal length even out (64 rows of up to 8192: 236 whole,
//    224 in two, 218 in four).
int attend_splits(int heads, const w4a8_kv_cache &c, const w4a8_kv_rows &r) {
    const int group = heads / c.kv_heads, each = attend_rows_each(group, r);
    const long groups = (long)((r.m + each - 1) / each) * c.kv_heads * ((group + HEADS - 1) / HEADS);
    const long rounds = ((long)r.table_pages * c.page_size + TILE * WAVES - 1) / (TILE * WAVES);
    if (rounds <= 3 || (rounds <= 8 && groups >= 192)) return 1;
    const auto least = [](long a, long b) { return a < b ? a : b; };
    const long full = least((512 + groups - 1) / groups, rounds);
    const long even = least((4096 + groups - 1) / groups, rounds / 16);
    return (int)least(full > even ? full : even, MAX_SPLITS);
}

// Whether K and V are loaded past the caches, by what the rows' tables may hold of them: a decode comes back to a layer's
// cache after all of the other layers' and the weights. From 8 MB on that is faster also where calls follow each other
// (a row of 4096 x 8 x 128 9.6 us against 10.1; 128 rows of 1024 88.9 against 98.9; two of 131072 x 8 x 64 88.4
// against 97.3), but for sizes that stay in the Infinity Cache then (64 MB 24.7 against 20.5). Below, what was appended
// or read last may still be there (1024 x 8 x 128 8.2 against 8.7).
bool attend_streams(const w4a8_kv_cache &c, const w4a8_kv_rows &r) {
    return r.table_stride != 0 && (double)r.m * r.table_pages * c.page_size * c.kv_heads * c.head_dim * 4.0 >= 8e6;
}

}  // namespace

size_t paged_attention_workspace_bytes(int heads, const w4a8_kv_cache &c, const w4a8_kv_rows &r) {
    const int splits = attend_splits(heads, c, r);
    return splits > 1 ? (size_t)r.m * heads * splits * (c.head_dim + 2) * sizeof(float) : 0;
}

hipError_t launch_paged_attention(const float *q, int heads, const w4a8_kv_cache &c, const w4a8_kv_rows &r, float scale,
                                  float *out, void *workspace, hipStream_t stream) {
    AttendArgs a{};
    a.q = q;
    a.k = c.k;
    a.v = c.v;
    a.table = r.table;
    a.table_stride = r.table_stride;
    a.table_pages = r.table_pages;
    a.pos = r.pos;
    a.m = r.m;
    a.out = out;
    a.heads = heads;
    a.group = heads / c.kv_heads;
    a.head_tiles = (a.group + HEADS - 1) / HEADS;
    a.rows_each = attend_rows_each(a.group, r);
    a.kv_heads = c.kv_heads;
    a.pages = c.pages;
    a.page_shift = __builtin_ctz((unsigned)c.page_size);
    a.splits = attend_splits(heads, c, r);
    if (a.splits > 1) {
        a.part = static_cast<float *>(workspace);
        a.part_ml = a.part + (size_t)r.m * heads * a.splits * c.head_dim;
    }
    a.scale = (float)((double)scale * 1.4426950408889634074);
    const unsigned grid = (unsigned)((long)((r.m + a.rows_each - 1) / a.rows_each) * a.kv_heads * a.head_tiles * a.splits);
    const auto go = [&](auto *kernel, auto *join) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * WAVES), 0, stream, a);
        if (a.splits > 1) {
            if (hipError_t e = hipGetLastError()) return e;
            hipLaunchKernelGGL(join, dim3((unsigned)(r.m * heads)), dim3(256), 0, stream, a);
        }
        return hipGetLastError();
    };
    const bool f16 = c.dtype == W4A8_KV_F16;
    const Reading how = a.rows_each > 1 ? SHARED : attend_streams(c, r) ? STREAMED : CACHED;
    const auto pick = [&](auto *cached, auto *streamed, auto *shared) {
        return how == SHARED ? shared : how == STREAMED ? streamed : cached;
    };
#define W4A8_ATTEND(D)                                                                                             \
    case D:                                                                                                        \
        return go(f16 ? pick(&attend_kernel<f16_t, D, CACHED>, &attend_kernel<f16_t, D, STREAMED>,                 \
                             &attend_kernel<f16_t, D, SHARED>)                                                     \
                      : pick(&attend_kernel<bf16_t, D, CACHED>, &attend_kernel<bf16_t, D, STREAMED>,               \
                             &attend_kernel<bf16_t, D, SHARED>),                                                   \
                  &attend_join_kernel<D>)
    switch (c.head_dim) {
        W4A8_ATTEND(64);
        W4A8_ATTEND(96);
        W4A8_ATTEND(128);
        W4A8_ATTEND(256);
        default: return hipErrorInvalidValue;
    }
#undef W4A8_ATTEND
}

}  // namespace w4a8
