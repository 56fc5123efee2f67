// Rope and the append to the paged cache (include/w4a8_step.h): what stands
// between the q|k|v GEMV and the attention (board/tp/tp_llama.cpp:835-856).
//
//   (a, b) -> (a cos - b sin, b cos + a sin), angle pos * inv_freq[pair].
//
// Bytes are the bound for a prompt (a row is read once, q written as float32,
// k and v as 16-bit values), latency for a decode. A thread takes eight values
// of a head (two float4 loads: the four pairs that it turns); a workgroup 256
// such items of one row, for which it takes the row's sines and cosines once,
// into LDS, while its loads are on their way. 1024 rows of 32 + 8 + 8 heads of
// 128 take 13.1 us, 6.1 TB/s; 2011 rows of heads of 64 9.3 us, 4.9 TB/s (two
// workgroups of 192 threads a row, each with the row's angles to take first);
// 64 rows of heads of 128 2.5 us.
#include "../../include/w4a8_step.h"
#include "kernels.h"
#include "kv_device.h"

namespace w4a8 {

namespace {

// sin and cos of pos * freq, within 2^-23 up to 2^40 radians. The product of a
// 31-bit integer and a float32 may take 55 bits: it is held as a float64 and what
// that leaves. Of both, what is left by the nearest multiple of pi / 2 (two
// float64, so to 2^-69 there) is taken: far positions are as exact as near ones.
// Then, |r| <= pi / 4, the series of both in float32, to r^9 and r^10 (the next
// terms are under 2^-29), what float32 left of r carried as `lo` through the
// first-order terms.
__device__ __forceinline__ void rope_angle(int pos, float freq, float &s, float &c) {
    const double a = (double)pos * (double)freq, rest = fma((double)pos, (double)freq, -a);
    const double n = rint(a * 0.63661977236758134308);           // 2 / pi
    const double r = fma(n, -6.1232339957367660359e-17, fma(n, -1.5707963267948965580, a)) + rest;
    const float hi = (float)r, lo = (float)(r - (double)hi);
    const float z = hi * hi;
    float p = fmaf(z, 1.0f / 362880, -1.0f / 5040);
    p = fmaf(z, p, 1.0f / 120);
    p = fmaf(z, p, -1.0f / 6);
    const float s0 = fmaf(hi * z, p, hi);
    p = fmaf(z, -1.0f / 3628800, 1.0f / 40320);
    p = fmaf(z, p, -1.0f / 720);
    p = fmaf(z, p, 1.0f / 24);
    p = fmaf(z, p, -0.5f);
    const float c0 = fmaf(z, p, 1.0f);
    const float s1 = fmaf(lo, c0, s0), c1 = fmaf(-lo, s0, c0);
    // n quarter turns; n mod 4 of a float64 that may pass 32 bits.
    const int quarter = (int)(n - 4.0 * floor(n * 0.25));
    const float x = quarter & 1 ? c1 : s1, y = quarter & 1 ? s1 : c1;
    s = quarter & 2 ? -x : x;
    c = (quarter + 1) & 2 ? -y : y;
}

struct AppendArgs {
    const float *qkv, *inv_freq;
    float *q_out;
    void *k, *v;
    const int32_t *table, *pos;
    int64_t table_stride;
    int heads, kv_heads, head_dim, rope_dim, pages, page_shift, table_pages, parts;
};

// The row's sines and cosines into LDS, for every thread after the barrier.
struct Turns {
    float sine[128], cosine[128];
};
__device__ __forceinline__ void turns_fill(const AppendArgs &a, int pos, Turns &t) {
    for (int i = threadIdx.x; i < a.rope_dim >> 1; i += blockDim.x) rope_angle(pos, a.inv_freq[i], t.sine[i], t.cosine[i]);
    __syncthreads();
}

__device__ __forceinline__ void turn(float &x, float &y, float s, float c) {
    const float u = fmaf(x, c, -(y * s)), v = fmaf(y, c, x * s);
    x = u;
    y = v;
}

// Rounded to nearest even, overflow to infinity.
template <class T>
__device__ __forceinline__ void store4(T *to, float4 f) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *reinterpret_cast<vec *>(to) = vec{(T)f.x, (T)f.y, (T)f.z, (T)f.w};
}
__device__ __forceinline__ void store4(float *to, float4 f) { *reinterpret_cast<float4 *>(to) = f; }

template <class T, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_append_kernel(AppendArgs a) {
    constexpr int ITEMS = D / 8;                     // of a head
    __shared__ Turns t;
    const int row = blockIdx.x / a.parts, item = (blockIdx.x % a.parts) * blockDim.x + threadIdx.x;
    const int pos = a.pos[row];
    const int head = item / ITEMS, j = item % ITEMS;
    const int all = a.heads + 2 * a.kv_heads;
    const bool works = head < all;
    // The item's two float4s, each beside the neighbours' in memory: the pairs (i, i + rope_dim / 2) of four i, or
    // (side by side, or nothing to turn) half a head apart; past a partial rope_dim, eight in a row.
    const bool ropes = head < a.heads + a.kv_heads;
    const bool halves = !INTERLEAVED && ropes;
    const bool turns = halves && 8 * j < a.rope_dim;
    const int d0 = halves && !turns ? 8 * j : 4 * j;
    const int d1 = turns ? 4 * j + (a.rope_dim >> 1) : halves ? 8 * j + 4 : 4 * j + D / 2;
    float4 x{}, y{};
    if (works && pos >= 0) {
        const float *src = a.qkv + ((size_t)row * all + head) * D;
        x = *reinterpret_cast<const float4 *>(src + d0);
        y = *reinterpret_cast<const float4 *>(src + d1);
    }
    if (pos >= 0) turns_fill(a, pos, t);             // the same in every thread of the workgroup
    if (!works) return;
    if (pos >= 0 && INTERLEAVED && ropes) {
        if (d0 < a.rope_dim) {
            turn(x.x, x.y, t.sine[d0 / 2], t.cosine[d0 / 2]);
            turn(x.z, x.w, t.sine[d0 / 2 + 1], t.cosine[d0 / 2 + 1]);
        }
        if (d1 < a.rope_dim) {
            turn(y.x, y.y, t.sine[d1 / 2], t.cosine[d1 / 2]);
            turn(y.z, y.w, t.sine[d1 / 2 + 1], t.cosine[d1 / 2 + 1]);
        }
    }
    if (pos >= 0 && turns) {
        turn(x.x, y.x, t.sine[d0], t.cosine[d0]);
        turn(x.y, y.y, t.sine[d0 + 1], t.cosine[d0 + 1]);
        turn(x.z, y.z, t.sine[d0 + 2], t.cosine[d0 + 2]);
        turn(x.w, y.w, t.sine[d0 + 3], t.cosine[d0 + 3]);
    }
    if (head < a.heads) {                            // an empty row's q: zeros
        float *to = a.q_out + ((size_t)row * a.heads + head) * D;
        store4(to + d0, x);
        store4(to + d1, y);
        return;
    }
    if (pos < 0) return;
    const int page = kv_page(a.table + row * a.table_stride, pos >> a.page_shift, a.table_pages, a.pages);
    if (page < 0) return;
    const int kvh = ropes ? head - a.heads : head - a.heads - a.kv_heads;
    const int slot = pos & ((1 << a.page_shift) - 1);
    T *to = static_cast<T *>(ropes ? a.k : a.v) + kv_offset(page, a.kv_heads, kvh, a.page_shift, D) + (size_t)slot * D;
    store4(to + d0, x);
    store4(to + d1, y);
}

// Any even rope_dim: a value a thread at a time, one workgroup a row.
template <class T>
__global__ __launch_bounds__(256) void rope_append_any_kernel(AppendArgs a, bool interleaved) {
    __shared__ Turns t;
    const int row = blockIdx.x, pos = a.pos[row], half = a.rope_dim >> 1, d_head = a.head_dim;
    float *qo = a.q_out + (size_t)row * a.heads * d_head;
    if (pos < 0) {
        for (int i = threadIdx.x; i < a.heads * d_head; i += 256) qo[i] = 0.0f;
        return;
    }
    const int page = kv_page(a.table + row * a.table_stride, pos >> a.page_shift, a.table_pages, a.pages);
    const int slot = pos & ((1 << a.page_shift) - 1);
    turns_fill(a, pos, t);
    const float *x = a.qkv + (size_t)row * (a.heads + 2 * a.kv_heads) * d_head;
    for (int i = threadIdx.x; i < (a.heads + 2 * a.kv_heads) * d_head; i += 256) {
        const int h = i / d_head, d = i - h * d_head;
        float y = x[i];
        if (h < a.heads + a.kv_heads && d < a.rope_dim) {
            const bool second = interleaved ? d & 1 : d >= half;
            const int pair = interleaved ? d >> 1 : second ? d - half : d, apart = interleaved ? 1 : half;
            float other = x[second ? i - apart : i + apart];
            if (second) {
                turn(other, y, t.sine[pair], t.cosine[pair]);
            } else {
                turn(y, other, t.sine[pair], t.cosine[pair]);
            }
        }
        if (h < a.heads) {
            qo[i] = y;
        } else if (page >= 0) {
            const bool is_k = h < a.heads + a.kv_heads;
            const int kvh = is_k ? h - a.heads : h - a.heads - a.kv_heads;
            static_cast<T *>(is_k ? a.k : a.v)[kv_offset(page, a.kv_heads, kvh, a.page_shift, d_head) +
                                               (size_t)slot * d_head + d] = (T)y;
        }
    }
}

}  // namespace

hipError_t launch_rope_append(const float *qkv, int heads, const w4a8_kv_cache &c, const w4a8_kv_rows &r,
                              const float *inv_freq, int rope_dim, bool interleaved, float *q_out, hipStream_t stream) {
    AppendArgs a{qkv, inv_freq, q_out, c.k, c.v, r.table, r.pos, r.table_stride, heads, c.kv_heads, c.head_dim, rope_dim,
                 c.pages, __builtin_ctz((unsigned)c.page_size), r.table_pages, 1};
    const bool f16 = c.dtype == W4A8_KV_F16;
    if (rope_dim % 8) {   // an item's pairs would not be whole float4s
        hipLaunchKernelGGL(f16 ? rope_append_any_kernel<f16_t> : rope_append_any_kernel<bf16_t>, dim3((unsigned)r.m),
                           dim3(256), 0, stream, a, interleaved);
        return hipGetLastError();
    }
    const int items = (heads + 2 * c.kv_heads) * (c.head_dim / 8);
    a.parts = (items + 255) / 256;
    const unsigned threads = (unsigned)((items + a.parts - 1) / a.parts + 63) / 64 * 64;
    const auto go = [&](auto *h1, auto *h0, auto *b1, auto *b0) {
        hipLaunchKernelGGL(f16 ? interleaved ? h1 : h0 : interleaved ? b1 : b0, dim3((unsigned)(r.m * a.parts)),
                           dim3(threads), 0, stream, a);
        return hipGetLastError();
    };
#define W4A8_APPEND(D)                                                                                    \
    case D:                                                                                               \
        return go(&rope_append_kernel<f16_t, D, true>, &rope_append_kernel<f16_t, D, false>,              \
                  &rope_append_kernel<bf16_t, D, true>, &rope_append_kernel<bf16_t, D, false>)
    switch (c.head_dim) {
        W4A8_APPEND(64);
        W4A8_APPEND(96);
        W4A8_APPEND(128);
        W4A8_APPEND(256);
        default: return hipErrorInvalidValue;
    }
#undef W4A8_APPEND
}

}  // namespace w4a8
