// q3t_kv8_kernels.h -- kernels of the 8-bit attention cache's operators
// (include/q3t_kv8.h): rotary positions, append, attention, eviction, read.
#pragma once

#include "../../include/q3t_kv8.h"
#include "q3t_numerics.h"

namespace q3t {
namespace kv8 {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;   // element types (ggml ids)
constexpr int kBlk = Q3T_KV8_BLOCK;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Elements 0 .. 7 from p, as fp32.  vec: p is 16-byte aligned.
template <int T>
__device__ __forceinline__ void load8(const void * base, int64_t at, bool vec, float (&x)[8]) {
    if constexpr (T == kF32) {
        const float * p = (const float *) base + at;
        if (vec) {
            const f4 a = *(const f4 *) p, b = *(const f4 *) (p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e];
        }
    } else {
        const uint16_t * p = (const uint16_t *) base + at;
        uint32_t w[4];
        if (vec) {
            const u4 v = *(const u4 *) p;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = p[2 * e] | (uint32_t) p[2 * e + 1] << 16;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = (uint16_t) (w[e / 2] >> (16 * (e & 1)));
            x[e] = T == kF16 ? h2f(h) : bf2f(h);
        }
    }
}

template <int T>
__device__ __forceinline__ void store8(void * base, int64_t at, bool vec, const float (&x)[8]) {
    if constexpr (T == kF32) {
        float * p = (float *) base + at;
        if (vec) {
            *(f4 *) p = (f4){x[0], x[1], x[2], x[3]};
            *(f4 *) (p + 4) = (f4){x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = x[e];
        }
    } else {
        uint16_t * p = (uint16_t *) base + at;
        uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = T == kF16 ? f2h(x[e]) : f2bf(x[e]);
        if (vec) {
            u4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = h[2 * e] | (uint32_t) h[2 * e + 1] << 16;
            *(u4 *) p = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = h[e];
        }
    }
}

template <class F>
__device__ __forceinline__ void by_type(int t, F f) {
    if (t == kF32) f(std::integral_constant<int, kF32>{});
    else if (t == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kBF16>{});
}

// ------------------------------------------------------------------ rotary
struct RopeRows {
    const void * x; void * y;
    int64_t xt, xh, yt, yh;
    const float * gain;
    int32_t n_head, xtype, ytype, vec;   // vec: every row 16-byte aligned on both sides
};
struct RopeArgs {
    RopeRows r[4];
    const int32_t * pos; const double * freq;
    int64_t n_tokens;
    int32_t pos0, head_dim, rot, inter;
    int32_t per;                         // tokens a workgroup
    float mscale, eps;
};

constexpr int kRopeT = 256;
constexpr int kRopeMax = 128;            // pairs a row at most
constexpr int kRopeTok = 8;              // tokens a workgroup at most

// grid (tokens / per, tensors).  A workgroup takes `per` tokens of one tensor:
// their sines and cosines first, then a row of D dims by a group of D / 16 lanes (to a
// power of two), 16 neighbouring dims a lane; a rotated dim's partner comes through
// LDS.
template <int XT, int YT>
__device__ __forceinline__ void rope_rows(const RopeArgs & a, const RopeRows & r, const float2 * cs, float * row_lds) {
    const int D = a.head_dim, half = a.rot / 2, lanes = (D + 15) / 16;
    int lpr = 1;
    while (lpr < lanes) lpr <<= 1;
    const int t = threadIdx.x, sub = t % lpr, grp = t / lpr, groups = kRopeT / lpr;
    const int64_t tok0 = (int64_t) blockIdx.x * a.per;
    const int nt = (int) min((int64_t) a.per, a.n_tokens - tok0), rows = nt * r.n_head;
    float * mine = row_lds + grp * D;
    const int d0 = sub * 16;
    for (int base = 0; base < rows; base += groups) {
        const int row = base + grp;
        const bool on = row < rows && sub < lanes;
        const int tok = row < rows ? row / r.n_head : 0, head = row < rows ? row % r.n_head : 0;
        float x[2][8] = {};
        if (on) {
            const int64_t at = (tok0 + tok) * r.xt + head * r.xh + d0;
            load8<XT>(r.x, at, r.vec, x[0]);
            load8<XT>(r.x, at + 8, r.vec, x[1]);
        }
        if (r.gain) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) ss = fmaf(x[e / 8][e % 8], x[e / 8][e % 8], ss);
            for (int m = 1; m < lpr; m <<= 1) ss += __shfl_xor(ss, m);
            const float rs = 1.0f / sqrtf(ss / (float) D + a.eps);
            if (on)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e / 8][e % 8] = x[e / 8][e % 8] * rs * r.gain[d0 + e];
        }
        if (on)
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[d0 + e] = x[e / 8][e % 8];
        __syncthreads();
        if (on) {
            const float2 * c = cs + tok * half;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = d0 + e;
                if (d >= a.rot) continue;
                const bool second = a.inter ? d & 1 : d >= half;
                const int i = a.inter ? d >> 1 : second ? d - half : d;
                const int other = a.inter ? d ^ 1 : second ? d - half : d + half;
                const float z = x[e / 8][e % 8], w = mine[other];
                x[e / 8][e % 8] = second ? z * c[i].x + w * c[i].y : z * c[i].x - w * c[i].y;
            }
            const int64_t at = (tok0 + tok) * r.yt + head * r.yh + d0;
            store8<YT>(r.y, at, r.vec, x[0]);
            store8<YT>(r.y, at + 8, r.vec, x[1]);
        }
        __syncthreads();
    }
}

// The angle pos * f in 64 bits, brought to [-pi, pi] by the nearest multiple of
// 2 pi (as the sum of two doubles: |pos * f| < 2^31 turns leave 2^-50), and its
// sine and cosine in fp32.
__device__ __forceinline__ float2 rope_angle(int pos, double f, float mscale) {
    const double a = (double) pos * f;
    const double n = rint(a * 0.15915494309189535);
    double r = fma(-n, 6.283185307179586, a);
    r = fma(-n, 2.4492935982947064e-16, r);
    float s, c;
    sincosf((float) r, &s, &c);
    return make_float2(c * mscale, s * mscale);
}

__global__ __launch_bounds__(kRopeT) void k_rope(RopeArgs a) {
    __shared__ float2 cs[kRopeTok * kRopeMax];
    __shared__ float rows[kRopeT * 16];
    const RopeRows r = a.r[blockIdx.y];
    const int64_t tok0 = (int64_t) blockIdx.x * a.per;
    const int nt = (int) min((int64_t) a.per, a.n_tokens - tok0), half = a.rot / 2;
    for (int i = threadIdx.x; i < nt * half; i += kRopeT) {
        const int64_t tok = tok0 + i / half;
        const int pos = (a.pos ? a.pos[tok] : (int) tok) + a.pos0;
        cs[i] = rope_angle(pos, a.freq[i % half], a.mscale);
    }
    __syncthreads();
    by_type(r.xtype, [&](auto xt) {
        by_type(r.ytype, [&](auto yt) { rope_rows<decltype(xt)::value, decltype(yt)::value>(a, r, cs, rows); });
    });
}

// ------------------------------------------------------------------ append
struct AppendArgs {
    q3t_kv8 c;
    const void * k, * v;
    int64_t xs, xr, xh;
    const int32_t * start, * n_new;
    int32_t start0, n_rows, type, vec;
};

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The code of x at scale s: x / s to the nearest even whole number.
__device__ __forceinline__ int code_of(float x, float s) {
    if (x != x || !(s > 0.0f)) return 0;
    return (int) fminf(fmaxf(rintf(x / s), -127.0f), 127.0f);
}

__device__ __forceinline__ u2 pack8(const int (&q)[8]) {
    u2 w = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= ((uint32_t) q[e] & 255u) << (8 * (e % 4));
    return w;
}
__device__ __forceinline__ int byte_of(uint32_t w, int e) { return (int) (int8_t) (w >> (8 * e)); }

// 8 codes moved from one scale to a larger one by r = old / new.
__device__ __forceinline__ u2 rescale8(u2 w, float r) {
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = (int) rintf((float) byte_of(w[e / 4], e % 4) * r);
    return pack8(q);
}

// grid (blocks a sequence's rows can touch, heads * 2, sequences); 2 D threads:
// one workgroup a block of 16 slots and K or V, 8 dims of a row a thread.
template <int D, int T>
__global__ __launch_bounds__(2 * D) void k_append(AppendArgs a) {
    __shared__ float part[2 * D / 64];
    const int t = threadIdx.x, r = t / (D / 8), d0 = t % (D / 8) * 8;
    const int head = blockIdx.y >> 1, is_v = blockIdx.y & 1, s = blockIdx.z;
    const int64_t start = (int64_t) (a.start ? a.start[s] : 0) + a.start0;
    const int n = a.n_new ? min(max(a.n_new[s], 0), a.n_rows) : a.n_rows;
    const int64_t blk = (start >> 4) + blockIdx.x;
    if (blk < 0 || blk >= a.c.n_slots / kBlk || blk * kBlk >= start + n) return;
    const int64_t i = blk * kBlk + r - start;          // the row of this thread's slot
    const bool fresh = i >= 0 && i < n;
    const bool begun = start > blk * kBlk;             // slots before start: only ever in the first block
    int8_t * codes = (is_v ? a.c.v : a.c.k) + s * a.c.seq + head * a.c.head + (blk * kBlk + r) * D + d0;
    float * scale = (is_v ? a.c.vs : a.c.ks) + s * a.c.scale_seq + head * a.c.scale_head + blk;
    float x[8] = {};
    if (fresh) load8<T>(is_v ? a.v : a.k, s * a.xs + i * a.xr + head * a.xh + d0, a.vec, x);
    u2 was = {0u, 0u};
    const bool held = begun && i < 0;
    if (held) was = *(const u2 *) codes;
    const float s0 = begun ? *scale : 0.0f;
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = finite_f(x[e]) ? fmaxf(m, fabsf(x[e])) : m;
    m = wave_max_f(m);
    if ((t & 63) == 0) part[t >> 6] = m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (int w = 1; w < 2 * D / 64; ++w) m = fmaxf(m, part[w]);
    const float s1 = fmaxf(s0, m / 127.0f);
    if (fresh) {
        int q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = code_of(x[e], s1);
        *(u2 *) codes = pack8(q);
        if (!is_v && a.c.acc && d0 == 0) a.c.acc[s * a.c.acc_seq + head * a.c.acc_head + blk * kBlk + r] = 0.0f;
    } else if (held && s1 > s0) {
        *(u2 *) codes = rescale8(was, s0 / s1);
    }
    if (t == 0) *scale = s1;
}

// --------------------------------------------------------------- attention
struct AttendArgs {
    q3t_kv8 c;
    const void * q; void * o;
    int64_t qs, qr, qh, os, orow, oh;
    const int32_t * lens, * n_new;
    int32_t len0, q_type, o_type, n_rows, n_head, group, max_len, causal, weights, qvec, ovec;
    float scale;
    float * ws;
};

__device__ __forceinline__ int seq_len(const AttendArgs & a, int s) {
    const int64_t n = (int64_t) (a.lens ? a.lens[s] : 0) + a.len0;
    return (int) min(max(n, (int64_t) 0), (int64_t) a.max_len);
}
__device__ __forceinline__ int seq_rows(const AttendArgs & a, int s) {
    return a.n_new ? min(max(a.n_new[s], 0), a.n_rows) : a.n_rows;
}
// slots that row i sees
__device__ __forceinline__ int row_limit(const AttendArgs & a, int len, int n, int i) {
    return a.causal ? max(len - n + i + 1, 0) : len;
}

// One row of one head a workgroup, grid (rows, heads, sequences): its scores to the workspace, their softmax, the
// value sum by D dims x 256 / D slot groups.  The scores stay as log2 of the
// probabilities for k_attend_acc.
template <int D>
__global__ __launch_bounds__(256) void k_attend_row(AttendArgs a) {
    __shared__ float q[D], red[8], part[256], top;
    const int t = threadIdx.x, i = blockIdx.x, h = blockIdx.y, s = blockIdx.z, g = h / a.group;
    const int len = seq_len(a, s), n = seq_rows(a, s);
    if (i >= n) return;
    const int lim = row_limit(a, len, n, i);
    float * sc = a.ws + (((int64_t) s * a.n_head + h) * a.n_rows + i) * a.max_len;
    const int8_t * kb = a.c.k + s * a.c.seq + g * a.c.head, * vb = a.c.v + s * a.c.seq + g * a.c.head;
    const float * ks = a.c.ks + s * a.c.scale_seq + g * a.c.scale_head, * vs = a.c.vs + s * a.c.scale_seq + g * a.c.scale_head;
    if (t < D) {
        const uint16_t x = ((const uint16_t *) a.q)[s * a.qs + i * a.qr + h * a.qh + t];
        q[t] = a.q_type == kF16 ? h2f(x) : bf2f(x);
    }
    __syncthreads();
    // the row under a power of two that brings its largest value to [1, 2): products with codes stay in range
    if (t < 64) {
        float big = 0.0f;
        for (int d = t; d < D; d += 64) big = fmaxf(big, fabsf(q[d]));
        big = wave_max_f(big);
        if (t == 0) top = finite_f(big) && big > 0.0f ? big : 1.0f;
    }
    __syncthreads();
    const int ex = ilogbf(top);
    if (t < D) q[t] = ldexpf(q[t], -ex);
    __syncthreads();
    const float scale = ldexpf(a.scale * 1.4426950408889634f, ex);
    float m = -INFINITY;
    for (int j = t; j < lim; j += 256) {
        float x = 0.0f;
        const u4 * p = (const u4 *) (kb + (int64_t) j * D);
        for (int c = 0; c < D / 16; ++c) {
            const u4 w = p[c];
#pragma unroll
            for (int e = 0; e < 16; ++e) x = fmaf((float) byte_of(w[e / 4], e % 4), q[16 * c + e], x);
        }
        x *= ks[j / kBlk] * scale;
        sc[j] = x;
        m = fmaxf(m, x);
    }
    m = wave_max_f(m);
    if ((t & 63) == 0) red[t >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f;
    for (int j = t; j < lim; j += 256) l += exp2f(sc[j] - m);
    l = (float) wave_sum_d((double) l);
    if ((t & 63) == 0) red[4 + (t >> 6)] = l;
    __syncthreads();
    l = red[4] + red[5] + red[6] + red[7];
    const float lse = m + log2f(l);
    for (int j = t; j < lim; j += 256) sc[j] -= lse;
    __syncthreads();
    float o = 0.0f;
    const int d = t % D;
    for (int j = t / D; j < lim; j += 256 / D) o = fmaf(exp2f(sc[j]) * vs[j / kBlk], (float) vb[(int64_t) j * D + d], o);
    part[t] = o;
    __syncthreads();
    if (t >= D) return;
#pragma unroll
    for (int w = 1; w < 256 / D; ++w) o += part[t + w * D];
    const int64_t at = s * a.os + i * a.orow + h * a.oh + t;
    if (a.o_type == kF32) ((float *) a.o)[at] = o;
    else ((uint16_t *) a.o)[at] = a.o_type == kF16 ? f2h(o) : f2bf(o);
}

// grid (slots / 256, kv heads, sequences): acc of a slot grows by its
// probabilities, rows then heads in order.
__global__ __launch_bounds__(256) void k_attend_acc(AttendArgs a) {
    const int j = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y, s = blockIdx.z;
    const int len = seq_len(a, s), n = seq_rows(a, s);
    if (j >= len || !n) return;
    float w = 0.0f;
    for (int i = 0; i < n; ++i) {
        if (j >= row_limit(a, len, n, i)) continue;
        for (int e = 0; e < a.group; ++e)
            w += exp2f(a.ws[(((int64_t) s * a.n_head + g * a.group + e) * a.n_rows + i) * a.max_len + j]);
    }
    a.c.acc[s * a.c.acc_seq + g * a.c.acc_head + j] += w;
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
    q3t_kv8 f, t;
    const int32_t * lens;
    int32_t len0, keep, sink, recent;
    int32_t * kept, * len_out;
};

constexpr int kEvT = 1024;

// An fp32 weight as an integer of the same order; -0 as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// grid (kv heads, sequences): the kept slots of one head.  The threshold (the
// want-th largest weight of the slots between sink and recent) is found a byte at a
// time from the top by counting; then one pass in slot order numbers the kept
// slots, of those at the threshold the first ones.
__global__ __launch_bounds__(kEvT) void k_evict_select(EvictArgs a) {
    __shared__ uint32_t hist[256], sums[kEvT / 64];
    __shared__ uint32_t pick[2];
    const int t = threadIdx.x, h = blockIdx.x, s = blockIdx.y;
    const int64_t want_len = (int64_t) (a.lens ? a.lens[s] : 0) + a.len0;
    const int len = (int) min(max(want_len, (int64_t) 0), (int64_t) a.f.n_slots), left = min(len, a.keep);
    int32_t * kept = a.kept + ((int64_t) s * a.f.n_kv_head + h) * a.keep;
    if (h == 0 && t == 0 && a.len_out) a.len_out[s] = left;
    for (int i = left + t; i < a.keep; i += kEvT) kept[i] = -1;
    if (len <= a.keep) {
        for (int i = t; i < left; i += kEvT) kept[i] = i;
        return;
    }
    const float * acc = a.f.acc + s * a.f.acc_seq + h * a.f.acc_head;
    const int lo = a.sink, hi = len - a.recent;     // len > keep >= sink + recent
    uint32_t want = (uint32_t) (a.keep - a.sink - a.recent), prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int i = lo + t; i < hi; i += kEvT) {
            const uint32_t k = order_of(acc[i]);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (t == 0) {
            uint32_t above = 0;
            int b = 255;
            while (b > 0 && above + hist[b] < want) above += hist[b--];
            pick[0] = (uint32_t) b;
            pick[1] = above;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= 255u << shift;
        want -= pick[1];
        __syncthreads();
    }
    // prefix: the threshold; want: how many slots at it are kept
    uint32_t over = 0, at = 0;                      // kept for sure, and at the threshold, so far
    for (int base = 0; base < len; base += kEvT) {
        const int i = base + t;
        uint32_t c = 0;
        if (i < len) {
            if (i < lo || i >= hi) c = 1u << 16;
            else {
                const uint32_t k = order_of(acc[i]);
                c = k > prefix ? 1u << 16 : k == prefix ? 1u : 0u;
            }
        }
        uint32_t in = c;                            // inclusive prefix sum of both counts (at most 1,024 each)
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t y = __shfl_up(in, m);
            if ((t & 63) >= m) in += y;
        }
        if ((t & 63) == 63) sums[t >> 6] = in;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int w = 0; w < kEvT / 64; ++w) {
            if (w < (t >> 6)) before += sums[w];
            all += sums[w];
        }
        in += before;
        const uint32_t o = over + (in >> 16), e = at + (in & 0xffffu);      // including this slot
        if (c >> 16) kept[o - 1 + min(e, want)] = i;
        else if (c && e <= want) kept[o + e - 1] = i;
        over += all >> 16;
        at += all & 0xffffu;
        __syncthreads();
    }
}

// grid (blocks of 16 kept slots, kv heads, sequences), 4 D threads: one block's
// codes, 16 bytes a thread (K's first), scales and weights.
template <int D>
__global__ __launch_bounds__(2 * D) void k_evict_move(EvictArgs a) {
    const int t = threadIdx.x, h = blockIdx.y, s = blockIdx.z, b = blockIdx.x;
    const int is_v = t / D, r = t % D / (D / 16), d0 = t % (D / 16) * 16;
    const int32_t * kept = a.kept + ((int64_t) s * a.f.n_kv_head + h) * a.keep;
    const float * fs = (is_v ? a.f.vs : a.f.ks) + s * a.f.scale_seq + h * a.f.scale_head;
    const int slot = b * kBlk + r, from = slot < a.keep ? kept[slot] : -1;
    if (kept[b * kBlk] < 0) return;
    const float s0 = from >= 0 ? fs[from / kBlk] : 0.0f;
    float s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlk; ++i) {
        const int o = b * kBlk + i < a.keep ? kept[b * kBlk + i] : -1;
        if (o >= 0) s1 = fmaxf(s1, fs[o / kBlk]);
    }
    if (r == 0 && d0 == 0) *((is_v ? a.t.vs : a.t.ks) + s * a.t.scale_seq + h * a.t.scale_head + b) = s1;
    if (from < 0) return;
    u4 w = *(const u4 *) ((is_v ? a.f.v : a.f.k) + s * a.f.seq + h * a.f.head + (int64_t) from * D + d0);
    if (s0 < s1) {
        const float ratio = s0 / s1;
        const u2 p = rescale8((u2){w[0], w[1]}, ratio), q = rescale8((u2){w[2], w[3]}, ratio);
        w = (u4){p[0], p[1], q[0], q[1]};
    }
    *(u4 *) ((is_v ? a.t.v : a.t.k) + s * a.t.seq + h * a.t.head + (int64_t) slot * D + d0) = w;
    if (!is_v && d0 == 0)
        a.t.acc[s * a.t.acc_seq + h * a.t.acc_head + slot] = a.f.acc[s * a.f.acc_seq + h * a.f.acc_head + from];
}

// -------------------------------------------------------------------- read
struct ReadArgs {
    q3t_kv8 c;
    const int32_t * start;
    int32_t start0, n_rows, type;
    void * k, * v;
};

// grid (values / 8 / 256 of one sequence and of K or V, K or V, sequences): 8 values a thread.
template <int D, int T>
__global__ __launch_bounds__(256) void k_read(ReadArgs a) {
    const int is_v = blockIdx.y, s = blockIdx.z, H = a.c.n_kv_head;
    void * out = is_v ? a.v : a.k;
    if (!out) return;
    const int64_t at = ((int64_t) blockIdx.x * 256 + threadIdx.x) * 8, per = (int64_t) a.n_rows * H * D;
    if (at >= per) return;
    const int d0 = (int) (at % D), h = (int) (at / D % H);
    const int64_t slot = (int64_t) (a.start ? a.start[s] : 0) + a.start0 + at / D / H;
    float x[8] = {};
    if (slot >= 0 && slot < a.c.n_slots) {
        const u2 w = *(const u2 *) ((is_v ? a.c.v : a.c.k) + s * a.c.seq + h * a.c.head + slot * D + d0);
        const float f = ((is_v ? a.c.vs : a.c.ks) + s * a.c.scale_seq + h * a.c.scale_head)[slot / kBlk];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float) byte_of(w[e / 4], e % 4) * f;
    }
    store8<T>(out, s * per + at, true, x);
}

}  // namespace kv8
}  // namespace q3t
