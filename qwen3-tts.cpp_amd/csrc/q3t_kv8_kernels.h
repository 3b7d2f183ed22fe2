// q3t_kv8_kernels.h -- kernels of the 8-bit attention cache's operators
// (include/q3t_kv8.h): rotary positions, append, attention, eviction, read.
// Times are one MI355X's, kernels alone; a large copy runs at 5.2 TB/s there
// and an 8192^3 fp16 library product at 1,160 TFLOP/s.
#pragma once

#include "../../include/q3t_kv8.h"
#include "q3t_numerics.h"

namespace q3t {
namespace kv8 {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;   // element types (ggml ids)
constexpr int kBlk = Q3T_KV8_BLOCK;
constexpr int kWhole = 8;            // tiles of 64 slots that k_attend_few takes in one workgroup

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
    int32_t per, n;                      // tokens a workgroup, tensors
    float mscale, eps;
};

constexpr int kRopeT = 256;
constexpr int kRopeMax = 128;            // pairs a row at most
constexpr int kRopeTok = 8;              // tokens a workgroup at most

// Rows of `nt` tokens of one tensor: a row by a group of lanes (D / 16 of them, to a power of two), 16 dims a lane.
// WHOLE: the lane's dims are 8 pairs (16 neighbours where interleaved, else 8 dims and the 8 half a rotation on; rot a
// multiple of 16), so they turn in registers.  Else it has 16 neighbours, and their partners come through LDS (a
// lane's 16 values 17 words apart, which spreads a wave's over the banks).
template <int XT, int YT, bool WHOLE>
__device__ __forceinline__ void rope_rows(const RopeArgs & a, const RopeRows & r, int64_t tok0, int nt, const float2 * cs,
                                          float * row_lds) {
    const int D = a.head_dim, half = a.rot / 2, lanes = D / 16;
    int lpr = 1;
    while (lpr < lanes) lpr <<= 1;
    const int t = threadIdx.x, sub = t % lpr, grp = t / lpr, groups = kRopeT / lpr, rows = nt * r.n_head;
    const bool turns = 16 * sub < a.rot;            // WHOLE: this lane's dims are rotated ones
    const int d0 = WHOLE && !a.inter && turns ? 8 * sub : 16 * sub;
    const int d1 = WHOLE && !a.inter && turns ? half + 8 * sub : 16 * sub + 8;
    float * mine = row_lds + grp * 17 * lpr;
    for (int base = 0; base < rows; base += groups) {
        const int row = base + grp;
        const bool on = row < rows && sub < lanes;
        const int tok = row < rows ? row / r.n_head : 0, head = row < rows ? row % r.n_head : 0;
        float x[2][8] = {};
        if (on) {
            const int64_t at = (tok0 + tok) * r.xt + head * r.xh;
            load8<XT>(r.x, at + d0, r.vec, x[0]);
            load8<XT>(r.x, at + d1, r.vec, x[1]);
        }
        if (r.gain) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) ss = fmaf(x[e / 8][e % 8], x[e / 8][e % 8], ss);
            for (int m = 1; m < lpr; m <<= 1) ss += __shfl_xor(ss, m);
            const float rs = 1.0f / sqrtf(ss / (float) D + a.eps);
            if (on)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e / 8][e % 8] = x[e / 8][e % 8] * rs * r.gain[(e < 8 ? d0 : d1) + e % 8];
        }
        const float2 * c = cs + tok * half;
        if constexpr (WHOLE) {
            if (turns) {
                c += 8 * sub;
                if (a.inter) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float & p = x[e / 4][2 * (e % 4)], & q = x[e / 4][2 * (e % 4) + 1];
                        const float y = p * c[e].x - q * c[e].y;
                        q = q * c[e].x + p * c[e].y;
                        p = y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float p = x[0][e], q = x[1][e];
                        x[0][e] = p * c[e].x - q * c[e].y;
                        x[1][e] = q * c[e].x + p * c[e].y;
                    }
                }
            }
        } else {
            if (on)
#pragma unroll
                for (int e = 0; e < 16; ++e) mine[17 * sub + e] = x[e / 8][e % 8];
            __syncthreads();
            if (on)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int d = 16 * sub + e;
                    if (d >= a.rot) continue;
                    const bool second = a.inter ? d & 1 : d >= half;
                    const int i = a.inter ? d >> 1 : second ? d - half : d;
                    const int other = a.inter ? d ^ 1 : second ? d - half : d + half;
                    const float z = x[e / 8][e % 8], y = mine[other + other / 16];
                    x[e / 8][e % 8] = second ? z * c[i].x + y * c[i].y : z * c[i].x - y * c[i].y;
                }
            __syncthreads();
        }
        if (on) {
            const int64_t at = (tok0 + tok) * r.yt + head * r.yh;
            store8<YT>(r.y, at + d0, r.vec, x[0]);
            store8<YT>(r.y, at + d1, r.vec, x[1]);
        }
    }
}

// The angle pos * f in 64 bits, brought to [-pi, pi] by the nearest multiple of
// 2 pi (as the sum of two doubles: |pos * f| < 2^31 turns leave 2^-50), and its
// sine and cosine in fp32.
__device__ __forceinline__ float2 rope_angle(int64_t pos, double f, float mscale) {
    const double a = (double) pos * f;
    const double n = rint(a * 0.15915494309189535);
    double r = fma(-n, 6.283185307179586, a);
    r = fma(-n, 2.4492935982947064e-16, r);
    float s, c;
    sincosf((float) r, &s, &c);
    return make_float2(c * mscale, s * mscale);
}

// Bound by memory: 11,301 tokens of 36 heads (208 MB) 39 us, 2,049 tokens of 24 heads from fp32 to fp16 (38 MB) 10
// us, one token 4.8 us.  All rows through LDS took 106, 20 and 5.6: words 16 apart in the banks, and the angles once
// a tensor.
// grid (tokens / per).  A workgroup takes `per` tokens: their sines and cosines once for all heads of all tensors,
// then the rows.
__global__ __launch_bounds__(kRopeT) void k_rope(RopeArgs a) {
    __shared__ float2 cs[kRopeTok * kRopeMax];
    __shared__ float rows[kRopeT * 17];
    const int64_t tok0 = (int64_t) blockIdx.x * a.per;
    const int nt = (int) min((int64_t) a.per, a.n_tokens - tok0), half = a.rot / 2;
    for (int i = threadIdx.x; i < nt * half; i += kRopeT) {
        const int64_t tok = tok0 + i / half;
        const int64_t pos = (a.pos ? a.pos[tok] : tok) + (int64_t) a.pos0;
        cs[i] = rope_angle(pos, a.freq[i % half], a.mscale);
    }
    __syncthreads();
    for (int x = 0; x < a.n; ++x) {
        const RopeRows & r = a.r[x];
        by_type(r.xtype, [&](auto xt) {
            by_type(r.ytype, [&](auto yt) {
                if (a.rot % 16 == 0) rope_rows<decltype(xt)::value, decltype(yt)::value, true>(a, r, tok0, nt, cs, rows);
                else rope_rows<decltype(xt)::value, decltype(yt)::value, false>(a, r, tok0, nt, cs, rows);
            });
        });
    }
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
// one workgroup a block of 16 slots and K or V, 8 dims of a row a thread, so that a block's maximum, the codes it
// held before and its new ones meet in one place and a block has one writer.  Bound by its chain of one load, the
// maximum over the block and the divisions: 2,049 rows of 8 heads (12.6 MB) 7.7 us, one row of 16 sequences 3.6.
template <int D, int T>
__global__ __launch_bounds__(2 * D) void k_append(AppendArgs a) {
    __shared__ float part[2 * D / 64];
    const int t = threadIdx.x, r = t / (D / 8), d0 = t % (D / 8) * 8;
    const int head = blockIdx.y >> 1, is_v = blockIdx.y & 1, s = blockIdx.z;
    const int64_t start = (int64_t) (a.start ? a.start[s] : 0) + a.start0;
    const int n = a.n_new ? min(max(a.n_new[s], 0), a.n_rows) : a.n_rows;
    const int64_t blk = (start >> 4) + blockIdx.x;
    if (!n || blk < 0 || blk >= a.c.n_slots / kBlk || blk * kBlk >= start + n) return;
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
    int64_t qs, qr, qhd, os, orow, oh;
    const int32_t * lens, * n_new;
    int32_t len0, q_type, o_type, n_rows, n_head, group, max_len, causal, weights, qvec, ovec;
    float scale, per_group;             // 1 / group
    int32_t split_tiles, n_split;       // 64-slot tiles a split
    int32_t row_tiles;                  // k_attend_tile: row tiles of a sequence and kv head
    int32_t units, most;                // .. workgroups that their slots are split over (0: not split), tiles at most
    int32_t row_blocks;                 // k_attend_join: workgroups of a sequence and kv head that take rows
    int32_t score_len, rows16;          // scores a row; rows to a multiple of 16
    // workspace, each where the call needs it: [seq][kv head][split][row][D]; [..][row]: maximum, sum; [seq][kv
    // head][row][score_len]; [seq][kv head][rows16][D]: q in fp16; [seq][kv head][rows16]: its factor, the row's
    // maximum, 1 / its sum
    float * part; float2 * stat; float * score; uint16_t * qh; f4 * rowq;
    int2 * split;                       // k_attend_tile: [seq][kv head][row tile]: its first split, how many
};

__device__ __forceinline__ int seq_len(const AttendArgs & a, int s) {
    const int64_t n = (int64_t) (a.lens ? a.lens[s] : 0) + a.len0;
    return (int) min(max(n, (int64_t) 0), (int64_t) a.max_len);
}
__device__ __forceinline__ int seq_rows(const AttendArgs & a, int s) {
    return a.n_new ? min(max(a.n_new[s], 0), a.n_rows) : a.n_rows;
}
// splits that a call's kernels gave `slots` slots: one writes its rows itself, several leave parts for k_attend_join
__device__ __forceinline__ int splits_of(const AttendArgs & a, int slots) {
    return ((slots + 63) / 64 + a.split_tiles - 1) / a.split_tiles;
}
// the token of row (token * group + head): rows are under 2^21 and tokens under 2^16, so that the product's error, 2^-23
// of it, is under half a row's part of a token
__device__ __forceinline__ int token_of(const AttendArgs & a, int row) {
    return (int) (((float) row + 0.5f) * a.per_group);
}
// where the row's values of a sequence and kv head are in q or out
__device__ __forceinline__ int64_t row_at(const AttendArgs & a, int row, int g, int64_t per_row, int64_t per_head) {
    const int tok = token_of(a, row);
    return tok * per_row + (g * a.group + row - tok * a.group) * per_head;
}
// slots that row i sees
__device__ __forceinline__ int row_limit(const AttendArgs & a, int len, int n, int i) {
    return a.causal ? max(len - n + i + 1, 0) : len;
}

// ----------------------------------------------- operands of attention
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// Codes as fp16.  A code's byte with its top bit turned, under the high byte
// 0x64, is the half 1024 + (code + 128); minus 1152 that is the code, exactly.
__device__ __forceinline__ uint32_t halves(uint32_t biased, uint32_t sel) {
    const h2v x = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, biased, sel));
    return __builtin_bit_cast(uint32_t, x + (h2v){(_Float16) -1152, (_Float16) -1152});
}
constexpr uint32_t kSelLo = 0x04010400u, kSelHi = 0x04030402u;   // bytes 0, 1 or 2, 3 of a word, each under 0x64
__device__ __forceinline__ h8v halves8(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const i4 v = {(int) halves(a, kSelLo), (int) halves(a, kSelHi), (int) halves(b, kSelLo), (int) halves(b, kSelHi)};
    return __builtin_bit_cast(h8v, v);
}
__device__ __forceinline__ f4 mfma32(h8v a, h8v b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
    const h2v v = {(_Float16) a, (_Float16) b};
    return __builtin_bit_cast(uint32_t, v);
}

// This lane's dims off + lo (c % 2) + hi (c / 2) .. + 7 of a row of q as they are, all loads at once (a choice of
// type or alignment at each would wait for each).
template <int D>
__device__ __forceinline__ void load_row(const AttendArgs & a, int64_t at, bool on, int off, int lo, int hi, u4 (&w)[D / 32]) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) w[c] = (u4){0u, 0u, 0u, 0u};
    if (!on) return;
    const uint16_t * p = (const uint16_t *) a.q + at + off;
    if (a.qvec) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) w[c] = *(const u4 *) (p + lo * (c & 1) + hi * (c >> 1));
    } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint16_t * y = p + lo * (c & 1) + hi * (c >> 1) + 2 * e;
                w[c][e] = y[0] | (uint32_t) y[1] << 16;
            }
    }
}

// That row as MFMA operands, with the sign of the scale: fp16 as it is; bfloat16 under the power of two that brings
// the row's largest value to [1, 2) (all bits of values down to 2^-14 of the largest).  Returns the factor of a
// product with it (not negative), NaN for a row that is not finite.
template <int D>
__device__ __forceinline__ float row_operand(const AttendArgs & a, const u4 (&w)[D / 32], h8v (&q)[D / 32]) {
    const bool half = a.q_type == kF16;
    us2 most = {0, 0};                          // the largest magnitudes of even and odd dims, as integers
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, w[c][e] & 0x7fff7fffu));
    int big = max((int) most[0], (int) most[1]);
    big = max(big, __shfl_xor(big, 16));
    big = max(big, __shfl_xor(big, 32));
    const float ok = big < (half ? 0x7c00 : 0x7f80) ? 0.0f : __uint_as_float(0x7fc00000u);
    const float scale = fabsf(a.scale) * 1.4426950408889634f;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    if (half) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) q[c] = __builtin_bit_cast(h8v, w[c] ^ (u4){flip, flip, flip, flip});
        return scale + ok;
    }
    const int ex = min(max(big >> 7, 1), 254) - 127;
    const float f = ldexpf(1.0f, -ex);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        i4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t u = w[c][e] ^ flip;
            v[e] = (int) pack_h(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f);
        }
        q[c] = __builtin_bit_cast(h8v, v);
    }
    return ldexpf(scale, ex) + ok;
}

// For k_attend_drawn: 16 rows from `row0` on, in fp16 as the operands they are (a lane's 16 bytes side by side), and
// the factors; zeros for rows past the last.
template <int D>
__device__ __forceinline__ void keep_rows(const AttendArgs & a, int64_t head, int row0, bool on, const h8v (&q)[D / 32], float qs) {
    if (!a.qh || row0 >= a.rows16) return;
    const int l = threadIdx.x & 63;
    const int64_t at = head * a.rows16 + row0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) *(h8v *) (a.qh + at * D + 512 * c + 8 * l) = q[c];
    if (l >= 16) return;
    if (on) a.rowq[at + l][0] = qs;
    else a.rowq[at + l] = (f4){0.f, 0.f, 0.f, 0.f};
}

template <int N>
__device__ __forceinline__ void store_out(const AttendArgs & a, int64_t at, const float (&y)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        if (a.o_type == kF32) {
            float * p = (float *) a.o + at + j;
            if (a.ovec) *(f4 *) p = (f4){y[j], y[j + 1], y[j + 2], y[j + 3]};
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = y[j + e];
        } else {
            uint16_t * p = (uint16_t *) a.o + at + j, h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = a.o_type == kF16 ? f2h(y[j + e]) : f2bf(y[j + e]);
            if (a.ovec) *(u2 *) p = (u2){h[0] | (uint32_t) h[1] << 16, h[2] | (uint32_t) h[3] << 16};
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = h[e];
        }
    }
}

// The row's maximum and the reciprocal of its sum (0 where it saw no slot).
__device__ __forceinline__ float inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ void keep_sum(const AttendArgs & a, int64_t at, float top, float sum) {
    a.rowq[at][1] = top == -INFINITY ? 0.0f : top;
    a.rowq[at][2] = inverse(sum);
}

// The larger of lanes 16 (32) apart, in both, by moves between rows of lanes.
__device__ __forceinline__ float max_rows(float x) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// A row's base of exponents follows its largest score only once that is more than this above it: a tile then needs
// no exchange between lanes and no rescaling as a rule, and 2^1.9 kPScale is still an fp16 number.
constexpr float kSlack = 1.9f;
// The largest value scale of blocks b0 .. b1 - 1 (all 64 lanes), at least 2^-110: kPScale over it is then finite, and
// smaller scales take the probabilities below kPScale, which costs bits from 2^-124 down.
__device__ __forceinline__ float top_scale(const float * vs, int b0, int b1, int lane) {
    float x = 0x1p-110f;
    for (int b = b0 + lane; b < b1; b += 64) x = fmaxf(x, vs[b]);
    return wave_max_f(x);
}
constexpr float kPScale = 16384.0f;    // probabilities enter the value product times this (fp16's normal range then ends at 2^-28)

// Rows of one kv head and sequence (n_new x group of them, 16 RT at most), grid (kv heads, splits, sequences), NW
// waves; workgroups go to the XCDs in turn, so heads come first and a sequence's splits are turned by its number: the
// first splits, the only ones of short sequences, spread over all XCDs (16 sequences of 128 to 32,768 slots: 150 us
// with splits first, 119 so, before a row's loads went out together).  A split is split_tiles tiles of 64 slots; the waves take its tiles in turn, each with
// its own running maximum m and sum, and join at the end.
//   - S^T = K . Q^T: 16 slots (A, codes straight from memory) by 16 rows (B) an MFMA of 32 dims.  Lane (i = l % 16, k
//     = l / 16) holds dims 64 c + 16 k .. + 15 of slot i, and after it the scores of slots 4k .. 4k + 3 of row i.
//   - O^T = V^T . P^T: those probabilities are the B operand where they lie, if the 32 slots of an MFMA are taken as
//     4k + e of one block of 16, then of the next; lane (i, k) then needs the codes of dims (D / 16) i .. of those
//     slots, which it reads as one piece of a row, and turns round by byte permutations while they become halves.
//     Row i's dims (D / 4) k .. are its outputs.
//   - Codes are exact in fp16; a key block's scale multiplies its scores, a value block's the probabilities, under
//     the largest value scale of the split (vref) and kPScale, so that they neither overflow nor lose bits.
//   - With several splits each (four waves) writes m, the sum and its unnormalised rows; k_attend_join puts them
//     together.  Eight waves take calls for up to kWhole tiles alone, and their weights too.
// Bound by memory: those 16 sequences (8 kv heads of 128, 2 rows each, 540 MB) at 4.5 TB/s; 131,001 slots of 4 kv
// heads of 64 (67 MB) 16 us; 2,049 slots of 8 kv heads 7.6, where it is the chain of a length, a tile and the waves'
// join.  The next tile's keys go out when this one's scores are formed, its values when this one's product is: two
// whole tiles in registers leave one wave a SIMD and take 135 us where this took 119; 3 waves a SIMD spill (300).
template <int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW) void k_attend_few(AttendArgs a) {
    constexpr int NC = D / 32, NJ = D / 16, LD = D + 4;
    constexpr bool whole = NW > 4;                  // the only split of its slots: it adds up their weights too
    __shared__ float mo[NW][16][LD], mm[NW][16], ml[NW][16];
    __shared__ float kept[whole ? 8 : 1][whole ? kWhole * 64 : 1], tops[8], invs[8];
    const bool scored = whole && a.weights && a.n_rows * a.group <= 8;
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, i = l & 15, k = l >> 4;
    const int g = blockIdx.x, s = blockIdx.z, split = (blockIdx.y + s) % a.n_split;
    const int len = seq_len(a, s), n = seq_rows(a, s), rows = n * a.group;
    const int tiles = (len + 63) / 64, t0 = split * a.split_tiles, t1 = min(t0 + a.split_tiles, tiles);
    if (!n || (split && t0 >= tiles)) return;
    const bool parts = splits_of(a, len) > 1;
    const int8_t * kb = a.c.k + s * a.c.seq + g * a.c.head, * vb = a.c.v + s * a.c.seq + g * a.c.head;
    const float * sb = (l & 4 ? a.c.vs : a.c.ks) + s * a.c.scale_seq + g * a.c.scale_head;
    const int last = len - 1, last_blk = last / kBlk;
    const int64_t hd = (int64_t) s * a.c.n_kv_head + g;
    float * sco = a.score ? a.score + hd * a.n_rows * a.group * a.score_len : nullptr;

    u4 kr[4][D / 64];
    uint32_t vr[16][NJ / 4];
    float sr;
    // rows past the last slot are the last slot's again; a scale past it is taken as 0 where it is used (a choice here
    // would wait for the load)
    auto fetch_k = [&](int tile) {
        const int8_t * p = kb + (int64_t) tile * 64 * D;
        const int left = last - tile * 64;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
                kr[b][c] = *(const u4 *) (p + (uint32_t) (min(16 * b + i, left) * D + 64 * c + 16 * k));
        sr = sb[min(tile * 4 + (l & 3), last_blk)];
    };
    auto fetch_v = [&](int tile) {
        const int8_t * p = vb + (int64_t) tile * 64 * D;
        const int left = last - tile * 64;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const uint32_t off = (uint32_t) (min(16 * (x / 4) + 4 * k + x % 4, left) * D + NJ * i);
            if constexpr (D == 128) {
                const u2 y = *(const u2 *) (p + off);
                vr[x][0] = y[0];
                vr[x][1] = y[1];
            } else {
                vr[x][0] = *(const uint32_t *) (p + off);
            }
        }
    };
    const int first = t0 + w;
    if (first < t1) {
        fetch_k(first);
        fetch_v(first);
    }
    h8v q[RT][NC];
    float qs[RT], m[RT], sum[RT];
    int lim[RT];
    f4 o[RT][NJ];
    u4 raw[RT][NC];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = min(16 * r + i, rows - 1);
        load_row<D>(a, s * a.qs + row_at(a, row, g, a.qr, a.qhd), 16 * r + i < rows, 16 * k, 8, 64, raw[r]);
    }
    const float vref = top_scale(a.c.vs + s * a.c.scale_seq + g * a.c.scale_head, 4 * t0, min(4 * t1, last_blk + 1), l);
    const float vscale = kPScale / vref;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = 16 * r + i;
        const bool on = row < rows;
        const int tok = token_of(a, row);
        qs[r] = row_operand<D>(a, raw[r], q[r]);
        if (split == 0 && w == 0) keep_rows<D>(a, hd, 16 * r, on, q[r], qs[r]);
        lim[r] = on ? row_limit(a, len, n, tok) : 0;
        m[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[r][j] = (f4){0.f, 0.f, 0.f, 0.f};
    }
    const int lim_all = row_limit(a, len, n, 0);    // slots that every row sees
    for (int tile = first; tile < t1; tile += NW) {
        f4 sc[RT][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int r = 0; r < RT; ++r) sc[r][b] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const h8v kf = halves8(kr[b][c / 2][2 * (c & 1)], kr[b][c / 2][2 * (c & 1) + 1]);
#pragma unroll
                for (int r = 0; r < RT; ++r) sc[r][b] = mfma32(kf, q[r][c], sc[r][b]);
            }
        }
        const int sl = __float_as_int(tile * 4 + (l & 3) <= last_blk ? sr : 0.0f);
        float ks[4], vs[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            ks[b] = __int_as_float(__builtin_amdgcn_readlane(sl, b));
            vs[b] = __int_as_float(__builtin_amdgcn_readlane(sl, 4 + b));
        }
        if (tile + NW < t1) fetch_k(tile + NW);
        h8v p[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                sc[r][b] *= ks[b] * qs[r];
                if (tile * 64 + 63 >= lim_all)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[r][b][e] = tile * 64 + 16 * b + 4 * k + e < lim[r] ? sc[r][b][e] : -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[r][b][e]);
            }
            if (whole && scored && i < rows)
#pragma unroll
                for (int b = 0; b < 4; ++b) *(f4 *) &kept[i][tile * 64 + 16 * b + 4 * k] = sc[r][b];
            if (!whole && sco && 16 * r + i < rows)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *(f4 *) (sco + (int64_t) (16 * r + i) * a.score_len + tile * 64 + 16 * b + 4 * k) = sc[r][b];
            if (__any(top > m[r] + kSlack)) {
                const float mn = fmaxf(m[r], max_rows(top)), move = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - mn);
                m[r] = mn;
                sum[r] *= move;
#pragma unroll
                for (int j = 0; j < NJ; ++j) o[r][j] *= move;
            }
            const float base = m[r] == -INFINITY ? 0.0f : m[r];
            float add[4];
            uint32_t pw[4][2];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float f = vs[b] * vscale;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_exp2f(sc[r][b][e] - base);
                add[b] = (x[0] + x[1]) + (x[2] + x[3]);
                pw[b][0] = pack_h(x[0] * f, x[1] * f);
                pw[b][1] = pack_h(x[2] * f, x[3] * f);
            }
            sum[r] += (add[0] + add[1]) + (add[2] + add[3]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const i4 v = {(int) pw[2 * u][0], (int) pw[2 * u][1], (int) pw[2 * u + 1][0], (int) pw[2 * u + 1][1]};
                p[r][u] = __builtin_bit_cast(h8v, v);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < NJ / 4; ++d) {
                uint32_t f[4][4];                   // dims 4d .. 4d + 3 of this lane: slots in pairs
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t w0 = vr[8 * u + 2 * x][d] ^ 0x80808080u, w1 = vr[8 * u + 2 * x + 1][d] ^ 0x80808080u;
                    const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
                    f[0][x] = halves(lo, kSelLo);
                    f[1][x] = halves(lo, kSelHi);
                    f[2][x] = halves(hi, kSelLo);
                    f[3][x] = halves(hi, kSelHi);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const i4 v = {(int) f[j][0], (int) f[j][1], (int) f[j][2], (int) f[j][3]};
#pragma unroll
                    for (int r = 0; r < RT; ++r) o[r][4 * d + j] = mfma32(__builtin_bit_cast(h8v, v), p[r][u], o[r][4 * d + j]);
                }
            }
        if (tile + NW < t1) fetch_v(tile + NW);
    }
    // the waves' rows under their common maximum, added in wave order
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        sum[r] += __shfl_xor(sum[r], 16);
        sum[r] += __shfl_xor(sum[r], 32);
        if (r) __syncthreads();
        if (k == 0) { mm[w][i] = m[r]; ml[w][i] = sum[r]; }
        __syncthreads();
        float top = mm[0][i];
#pragma unroll
        for (int x = 1; x < NW; ++x) top = fmaxf(top, mm[x][i]);
        const float base = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m[r] - base) * (vref / kPScale);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < NJ; j += 4)
                *(f4 *) &mo[w][i][(D / 4) * k + NJ * e + j] = (f4){o[r][j][e], o[r][j + 1][e], o[r][j + 2][e], o[r][j + 3][e]} * f;
        __syncthreads();
        const int row = t >> 4, d0 = (t & 15) * NJ, at = 16 * r + row;
        if (row < 16 && at < rows) {
            float big = mm[0][row], all = 0.0f;
#pragma unroll
            for (int x = 1; x < NW; ++x) big = fmaxf(big, mm[x][row]);
#pragma unroll
            for (int x = 0; x < NW; ++x) all += ml[x][row] * __builtin_amdgcn_exp2f(mm[x][row] - (big == -INFINITY ? 0.0f : big));
            const int64_t cell = (hd * a.n_split + split) * a.n_rows * a.group + at;
            if (a.stat && d0 == 0) a.stat[cell] = make_float2(big, all);
            if (a.rowq && !parts && d0 == 0) keep_sum(a, hd * a.rows16 + at, big, all);
            if (scored && d0 == 0) {
                tops[row] = big == -INFINITY ? 0.0f : big;
                invs[row] = inverse(all);
            }
            const float inv = parts ? 1.0f : inverse(all);
            float y[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                y[j] = mo[0][row][d0 + j];
#pragma unroll
                for (int x = 1; x < NW; ++x) y[j] += mo[x][row][d0 + j];
                y[j] *= inv;
            }
            if (parts) {
#pragma unroll
                for (int j = 0; j < NJ; j += 4)
                    *(f4 *) (a.part + cell * D + d0 + j) = (f4){y[j], y[j + 1], y[j + 2], y[j + 3]};
            } else {
                store_out<NJ>(a, s * a.os + row_at(a, at, g, a.orow, a.oh) + d0, y);
            }
        }
    }
    if (scored) {
        __syncthreads();
        float * acc = a.c.acc + s * a.c.acc_seq + g * a.c.acc_head;
        for (int j = t; j < len; j += 64 * NW) {
            float add = 0.0f;
            for (int r = 0; r < rows; ++r)
                if (kept[r][j] != -INFINITY) add = fmaf(__builtin_amdgcn_exp2f(kept[r][j] - tops[r]), invs[r], add);
            acc[j] += add;
        }
    }
}

constexpr int kSplitMax = 1024;
constexpr int kTileT = 256, kTileRows = 128, kUnits = 512, kLeast = 4;

// acc of 1,024 slots (the blk-th) from the scores that k_attend_few kept; eight rows at most.
__device__ __forceinline__ void scored_slots(const AttendArgs & a, int blk) {
    __shared__ float2 row_sum[8];                   // a row's maximum and the reciprocal of its sum
    const int t = threadIdx.x, g = blockIdx.y, s = blockIdx.z;
    const int len = seq_len(a, s), n = seq_rows(a, s), rows = n * a.group, all_rows = a.n_rows * a.group;
    const int live = splits_of(a, len);
    const int64_t hd = (int64_t) s * a.c.n_kv_head + g;
    const int j = blk * 1024 + 4 * t;               // this thread's four slots
    if (blk * 1024 >= len || !n) return;
    const float * sco = a.score + hd * all_rows * a.score_len + min(j, a.score_len - 4);
    float * acc = a.c.acc + s * a.c.acc_seq + g * a.c.acc_head + j;
    f4 x[8], old = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < rows) x[r] = *(const f4 *) (sco + (int64_t) r * a.score_len);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < len) old[e] = acc[e];
    for (int r = t >> 6; r < rows; r += 4) {        // one wave a row
        const int64_t cell = hd * a.n_split * all_rows + r;
        float top = -INFINITY, sum = 0.0f;
        for (int y = t & 63; y < live; y += 64) top = fmaxf(top, a.stat[cell + (int64_t) y * all_rows].x);
        top = wave_max_f(top);
        const float base = top == -INFINITY ? 0.0f : top;
        for (int y = t & 63; y < live; y += 64) {
            const float2 st = a.stat[cell + (int64_t) y * all_rows];
            sum = fmaf(st.y, __builtin_amdgcn_exp2f(st.x - base), sum);
        }
#pragma unroll
        for (int y = 1; y < 64; y <<= 1) sum += __shfl_xor(sum, y);
        if ((t & 63) == 0) row_sum[r] = make_float2(base, inverse(sum));
    }
    __syncthreads();
    f4 add = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < rows)
#pragma unroll
            for (int e = 0; e < 4; ++e)             // a slot that the row does not see: unchanged, whatever the row's sum is
                if (x[r][e] != -INFINITY) add[e] = fmaf(__builtin_amdgcn_exp2f(x[r][e] - row_sum[r].x), row_sum[r].y, add[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < len) acc[e] = old[e] + add[e];
}

// The rows of all splits put together, grid (rows / rows a workgroup, then 1,024 slots' weights each where scores
// were kept; kv heads; sequences): D / 4 lanes a split, many splits of one row (MANY) by 1024 / D groups whose sums
// are added in order, or a row a group.
// Bound by the splits' rows (512 bytes each): 4,098 rows of 8 kv heads in up to 3 splits 8 us, 2 rows of 128
// (sequence, head)s and their weights (34 MB of scores and sums) 12.5, 8 rows in 256 splits 5.
template <int D, bool MANY>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a) {
    constexpr int LN = D / 4, GR = 256 / LN;
    __shared__ f4 po[GR][LN];
    __shared__ float fac[MANY ? kSplitMax : 1], red[8];
    if ((int) blockIdx.x >= a.row_blocks) return scored_slots(a, blockIdx.x - a.row_blocks);
    const int t = threadIdx.x, g = blockIdx.y, s = blockIdx.z, gr = t / LN, ln = t % LN;
    const int len = seq_len(a, s), n = seq_rows(a, s), rows = n * a.group, all_rows = a.n_rows * a.group;
    const int64_t hd = (int64_t) s * a.c.n_kv_head + g;
    const int row = MANY ? blockIdx.x : blockIdx.x * GR + gr;
    if (row >= rows) return;                        // MANY: the whole workgroup
    int live, step;                                 // splits, and how many rows of the workspace they are apart
    int64_t cell;
    if (a.row_tiles) {
        const int2 z = a.split[hd * a.row_tiles + row / kTileRows];
        live = z.y;
        step = a.c.n_kv_head * kTileRows;
        cell = ((int64_t) z.x * a.c.n_kv_head + g) * kTileRows + row % kTileRows;
    } else {
        live = splits_of(a, len);
        step = all_rows;
        cell = hd * a.n_split * all_rows + row;
    }
    if (live <= 1) return;                          // written by its split
    float top = -INFINITY, sum = 0.0f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    if constexpr (MANY) {
        for (int x = t; x < live; x += 256) top = fmaxf(top, a.stat[cell + (int64_t) x * step].x);
        top = wave_max_f(top);
        if ((t & 63) == 0) red[t >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float base = top == -INFINITY ? 0.0f : top;
        for (int x = t; x < live; x += 256) {
            const float2 st = a.stat[cell + (int64_t) x * step];
            fac[x] = __builtin_amdgcn_exp2f(st.x - base);
            sum = fmaf(st.y, fac[x], sum);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        if ((t & 63) == 0) red[4 + (t >> 6)] = sum;
        __syncthreads();
        sum = (red[4] + red[5]) + (red[6] + red[7]);
#pragma unroll 4
        for (int x = gr; x < live; x += GR) o += *(const f4 *) (a.part + (cell + (int64_t) x * step) * D + 4 * ln) * fac[x];
        po[gr][ln] = o;
        __syncthreads();
        if (gr) return;
#pragma unroll
        for (int x = 1; x < GR; ++x) o += po[x][ln];
    } else {
        // four splits' loads at once; the maximum so far moves with each four
        for (int x = 0; x < live; x += 4) {
            float2 st[4];
            f4 y[4];
            float most = top;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = cell + (int64_t) min(x + u, live - 1) * step;
                st[u] = a.stat[at];
                y[u] = *(const f4 *) (a.part + at * D + 4 * ln);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) most = fmaxf(most, st[u].x);
            const float base = most == -INFINITY ? 0.0f : most, move = __builtin_amdgcn_exp2f(top - base);
            o *= move;
            sum *= move;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float f = x + u < live ? __builtin_amdgcn_exp2f(st[u].x - base) : 0.0f;
                o += y[u] * f;
                sum = fmaf(st[u].y, f, sum);
            }
            top = most;
        }
    }
    if (a.rowq && ln == 0) keep_sum(a, hd * a.rows16 + row, top, sum);
    o *= inverse(sum);
    const float y[4] = {o[0], o[1], o[2], o[3]};
    store_out<4>(a, s * a.os + row_at(a, row, g, a.orow, a.oh) + 4 * ln, y);
}

// ----------------------------------------------- attention of many rows
// Which sequence, row tile and split of it workgroup blockIdx.x takes (heads are fastest); false: none.  Lengths are on
// the device, so the splits are chosen here, by every wave alike: of 63 lengths from the mean (kLeast tiles at least) on, 1/16
// octave apart, the shortest with which all row tiles of all sequences make no more than `units` workgroups, or none,
// and a row tile's splits of one length.  z: a wave's 512 ints of LDS, so many row tiles of sequences at most.
__device__ __forceinline__ bool find_split(const AttendArgs & a, int * z, int & s, int & row_tile, int & split, int & splits) {
    const int l = threadIdx.x & 63, seqs = a.c.n_seq, n_tile = seqs * a.row_tiles, me = blockIdx.x / a.c.n_kv_head;
    float all = 0.0f;
    for (int p = l; p < (n_tile + 7) / 8 * 8; p += 64) {
        int tiles = 0;
        if (p < n_tile) {
            const int sq = p % seqs, row0 = (a.row_tiles - 1 - p / seqs) * kTileRows, n = seq_rows(a, sq), rows = n * a.group;
            const int lim = row_limit(a, seq_len(a, sq), n, token_of(a, min(row0 + kTileRows, rows) - 1));
            if (row0 < rows) tiles = max(lim + 63, 64) / 64;
        }
        z[p] = tiles;
        all += (float) tiles;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) all += __shfl_xor(all, m);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    auto count = [](int tiles, float inv) { return (int) ceilf((float) tiles * inv); };
    const float mean = fmaxf(all * a.c.n_kv_head / a.units, (float) kLeast);
    const float inv = l == 63 ? 0.5f / a.most : 1.0f / (mean * __builtin_amdgcn_exp2f(l / 16.0f));
    int n = 0;
    for (int p = 0; p < n_tile; p += 8) {           // zeros behind the last
        const i4 x = *(const i4 *) (z + p), y = *(const i4 *) (z + p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) n += count(x[e], inv) + count(y[e], inv);
    }
    const float best = __shfl(inv, __builtin_ctzll(__ballot(n * a.c.n_kv_head <= a.units)));
    int own = 0, c[8], at[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        at[e] = own;
        c[e] = 8 * l + e < n_tile ? count(z[8 * l + e], best) : 0;
        own += c[e];
    }
    int in = own;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int y = __shfl_up(in, m);
        if (l >= m) in += y;
    }
    const uint64_t past = __ballot(in > me);
    if (!past) return false;
    const int lane = __builtin_ctzll(past), rest = me - (in - own);
    int p = 0;
    split = splits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (rest >= at[e] && rest < at[e] + c[e]) { p = 8 * l + e; split = rest - at[e]; splits = c[e]; }
    p = __builtin_amdgcn_readlane(p, lane);
    split = __builtin_amdgcn_readlane(split, lane);
    splits = __builtin_amdgcn_readlane(splits, lane);
    s = p % seqs;
    row_tile = a.row_tiles - 1 - p / seqs;
    return true;
}

// A tile of 128 rows (n_new x group of a sequence and kv head) over a split of its slots, grid (splits as find_split
// deals them, or heads and sequences, then row tiles; a head's workgroups share an XCD's L2), four
// waves of 32 rows.  Tiles of 64 slots become fp16 in LDS once for all rows.  Products, softmax and scales as in
// k_attend_few; here all waves go through the same tiles, with dims in their own order:
//   K in LDS: [slot][dim] in 16-byte chunks, chunk c of slot t at c ^ (t % (D / 8));
//   V in LDS: [dim][8 chunks], chunk 4u + k = slots 32u + 4k + e, then 32u + 16 + 4k + e (an operand of the value
//   product as it is), at chunk ^ f(dim) with f = (dim / 4) % 8 ^ 2 (dim % 4), so that both the 16 dims of a read and
//   the 32 dim quads of a write spread over all banks.
// Two buffers of each: the next tile's codes are on their way from memory while this one's products run, and go to
// LDS at the end, one barrier a tile.  A wave reads its operands from LDS four at a time, the next four before the
// MFMAs of these: left to itself the compiler waits for each read alone.
// Bound by issue: a wave and tile of 64 MFMAs (1,000 clocks) has 380 vector instructions (1,900 clocks: 32
// exponentials, 5 more instructions a score, 100 to turn codes into halves); alone on its SIMD it takes 4,000 clocks,
// two overlap to 2,500 each.  Beside the tiles a workgroup takes 12,000 clocks, 5 us: its place and length, q, its
// rows' way out.  2,049 rows over their own slots, 8 x 2 heads of 128 (17 GFLOP) 48 us and 8 for the join; 3 x 209
// rows over 4,001 to 12,011 slots (41 GFLOP) 85 us, 104 with splits of one length for all sequences, as long as the
// longest would need.  Measured and not kept: eight waves of 16 rows (115 us where this took 104: operands are read
// twice as often, and it spills), exponents with the scales folded in (3% faster, but scores past 2^16 then need a
// second form), the next tile's scores beside this tile's exponentials (124: no registers left for operand reads),
// wave priorities (no change).
template <int D>
__global__ __launch_bounds__(kTileT, 2) void k_attend_tile(AttendArgs a) {
    constexpr int RT = 2, NC = D / 32, NJ = D / 16, NCH = D / 8, KT = 64 * D;
    __shared__ __align__(16) uint16_t lds[4 * KT];      // K of even and odd tiles, V of even and odd tiles
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, i = l & 15, k = l >> 4;
    const int heads = a.c.n_kv_head, g = blockIdx.x % heads;
    int s = blockIdx.x / heads, row_tile = a.row_tiles - 1 - blockIdx.y, split = 0, splits = 1;
    if (a.units) {
        if (!find_split(a, (int *) lds + 512 * w, s, row_tile, split, splits)) return;
        __syncthreads();                            // the tiles go where lengths were
    }
    const int len = seq_len(a, s), n = seq_rows(a, s), rows = n * a.group, row0 = row_tile * kTileRows;
    if (row0 >= rows) return;
    const int64_t hd = (int64_t) s * heads + g;
    const int tiles = (row_limit(a, len, n, token_of(a, min(row0 + kTileRows, rows) - 1)) + 63) / 64;
    const int t0 = (int) ((int64_t) split * tiles / splits), t1 = (int) ((int64_t) (split + 1) * tiles / splits);
    const bool parts = splits > 1;
    if (a.units && split == 0 && t == 0)
        a.split[hd * a.row_tiles + row_tile] = make_int2((int) blockIdx.x / heads, splits);
    const bool work = row0 + 16 * RT * w < rows;        // this wave has rows

    const int plain = row_limit(a, len, n, token_of(a, row0)) / 64;    // tiles before this one need no mask
    const int last = len - 1, last_blk = last / kBlk;

    // staging: 32 bytes of a K row, and 4 dims of 8 V rows a thread; of 64 dims half the threads each
    const bool do_k = D == 128 || t >= 128, do_v = D == 128 || t < 128;
    const int kt = D == 128 ? t >> 2 : (t & 127) >> 1, kp = D == 128 ? t & 3 : t & 1;
    const int vq = t & (D / 4 - 1), vc = (D == 128 ? t : t & 127) / (D / 4);
    const int8_t * kb = a.c.k + s * a.c.seq + g * a.c.head, * vb = a.c.v + s * a.c.seq + g * a.c.head;
    const float * sb = (l & 4 ? a.c.vs : a.c.ks) + s * a.c.scale_seq + g * a.c.scale_head;
    u4 kr[2];
    uint32_t vr[8];
    float sr = 0.0f;
    // tiles past the split's end are its last one again, rows past the last slot the last slot's
    auto fetch_k = [&](int tile) {
        if (!do_k) return;
        tile = min(tile, t1 - 1);
        const int8_t * p = kb + (int64_t) tile * 64 * D;
        const uint32_t off = (uint32_t) (min(kt, last - tile * 64) * D + 32 * kp);
        kr[0] = *(const u4 *) (p + off);
        kr[1] = *(const u4 *) (p + off + 16);
    };
    auto fetch_v = [&](int tile) {
        tile = min(tile, t1 - 1);
        sr = sb[min(tile * 4 + (l & 3), last_blk)];
        if (!do_v) return;
        const int8_t * p = vb + (int64_t) tile * 64 * D;
        const int left = last - tile * 64;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            vr[e] = *(const uint32_t *) (p + (uint32_t) (min(32 * (vc >> 2) + 16 * (e >> 2) + 4 * (vc & 3) + (e & 3), left) * D + 4 * vq));
    };
    auto stash_k = [&](int tile) {
        if (!do_k) return;
        uint16_t * d = lds + (tile & 1) * KT + kt * D;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *(h8v *) (d + (((4 * kp + c) ^ (kt & (NCH - 1))) << 3)) = halves8(kr[c / 2][2 * (c & 1)], kr[c / 2][2 * (c & 1) + 1]);
    };
    auto stash_v = [&](int tile) {
        if (!do_v) return;
        uint16_t * d = lds + (2 + (tile & 1)) * KT + 4 * vq * 64;
        uint32_t f[4][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t w0 = vr[2 * x] ^ 0x80808080u, w1 = vr[2 * x + 1] ^ 0x80808080u;
            const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400u), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
            f[0][x] = halves(lo, kSelLo);
            f[1][x] = halves(lo, kSelHi);
            f[2][x] = halves(hi, kSelLo);
            f[3][x] = halves(hi, kSelHi);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(u4 *) (d + j * 64 + ((vc ^ (vq & 7) ^ (2 * j)) << 3)) = (u4){f[j][0], f[j][1], f[j][2], f[j][3]};
    };
    if (t0 < t1) {
        fetch_k(t0);
        fetch_v(t0);
    }
    h8v q[RT][NC];
    float qs[RT], m[RT], sum[RT];
    int lim[RT];
    f4 o[RT][NJ];
    u4 raw[RT][NC];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = row0 + 16 * (RT * w + r) + i, there = min(row, rows - 1);
        load_row<D>(a, s * a.qs + row_at(a, there, g, a.qr, a.qhd), row < rows, 8 * k, 32, 64, raw[r]);
    }
    const float vref = top_scale(a.c.vs + s * a.c.scale_seq + g * a.c.scale_head, 4 * t0, min(4 * t1, last_blk + 1), l);
    const float vscale = kPScale / vref;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = row0 + 16 * (RT * w + r) + i;
        const bool on = row < rows;
        const int tok = token_of(a, row);
        qs[r] = row_operand<D>(a, raw[r], q[r]);
        if (split == 0) keep_rows<D>(a, hd, row - i, on, q[r], qs[r]);
        lim[r] = on ? row_limit(a, len, n, tok) : 0;
        m[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[r][j] = (f4){0.f, 0.f, 0.f, 0.f};
    }
    auto step = [&](int tile, auto masked) {
        const int sl = __float_as_int(tile * 4 + (l & 3) <= last_blk ? sr : 0.0f);
        fetch_k(tile + 1);
        fetch_v(tile + 1);
        float ks[4], vs[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            ks[b] = __int_as_float(__builtin_amdgcn_readlane(sl, b));
            vs[b] = __int_as_float(__builtin_amdgcn_readlane(sl, 4 + b));
        }
        if (work) {
            const uint16_t * kd = lds + (tile & 1) * KT + i * D, * vd = lds + (2 + (tile & 1)) * KT + i * 64;
            f4 sc[RT][4];
            h8v kf[2][4];
            auto read_k = [&](int c) {
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    kf[c & 1][b] = *(const h8v *) (kd + 16 * b * D + (((4 * c + k) ^ (i & (NCH - 1))) << 3));
                __builtin_amdgcn_sched_barrier(0);
            };
            read_k(0);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (c + 1 < NC) read_k(c + 1);
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int r = 0; r < RT; ++r) sc[r][b] = mfma32(kf[c & 1][b], q[r][c], c ? sc[r][b] : (f4){0.f, 0.f, 0.f, 0.f});
            }
            bool grows = false;
            float top[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                // scaled and rounded before the maximum is taken, so that none is above it however large they are
                top[r] = -INFINITY;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    sc[r][b] *= ks[b] * qs[r];
                    if constexpr (decltype(masked)::value)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sc[r][b][e] = tile * 64 + 16 * b + 4 * k + e < lim[r] ? sc[r][b][e] : -INFINITY;
                    top[r] = fmaxf(top[r], fmaxf(fmaxf(sc[r][b][0], sc[r][b][1]), fmaxf(sc[r][b][2], sc[r][b][3])));
                }
                grows |= top[r] > m[r] + kSlack;
            }
            if (__any(grows)) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float mn = fmaxf(m[r], max_rows(top[r]));
                    const float move = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - mn);
                    m[r] = mn;
                    sum[r] *= move;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) o[r][j] *= move;
                }
            }
            // chunk 4u + k of dim 16 j + i: at (4 (u ^ j % 2) + k) ^ (i / 4) ^ 2 (i % 4)
            const int x0 = (k ^ (i >> 2) ^ (2 * (i & 3))) << 3;
            h8v vf[2][4];                           // of two dim tiles: u 0 of both, u 1 of both
            auto read_v = [&](int j) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    vf[(j / 2) & 1][x] = *(const h8v *) (vd + 16 * (j + (x & 1)) * 64 + (x0 ^ (32 * ((x >> 1) ^ (x & 1)))));
                __builtin_amdgcn_sched_barrier(0);
            };
            read_v(0);
            h8v p[RT][2];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
                uint32_t pw[4][2];
                float add = 0.0f;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float f = vs[b] * vscale;
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_exp2f(sc[r][b][e] - base);
                    add += (x[0] + x[1]) + (x[2] + x[3]);
                    pw[b][0] = pack_h(x[0] * f, x[1] * f);
                    pw[b][1] = pack_h(x[2] * f, x[3] * f);
                }
                sum[r] += add;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const i4 v = {(int) pw[2 * u][0], (int) pw[2 * u][1], (int) pw[2 * u + 1][0], (int) pw[2 * u + 1][1]};
                    p[r][u] = __builtin_bit_cast(h8v, v);
                }
            }
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                if (j + 2 < NJ) read_v(j + 2);
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int r = 0; r < RT; ++r) o[r][j + (x & 1)] = mfma32(vf[(j / 2) & 1][x], p[r][x >> 1], o[r][j + (x & 1)]);
            }
        }
        stash_k(tile + 1);
        stash_v(tile + 1);
        __syncthreads();
    };
    if (t0 < t1) {
        stash_k(t0);
        stash_v(t0);
        __syncthreads();
        int tile = t0;
        for (; tile < min(t1, plain); ++tile) step(tile, std::false_type{});
        for (; tile < t1; ++tile) step(tile, std::true_type{});
    }
    // rows to memory by way of LDS (fp32, 16-byte chunks c of row x at c ^ x; each wave its own 32 rows), 8 dims of a
    // row a thread: written from where they are they took 4 us, in a choice of type and alignment for each four dims
    float * mine = (float *) lds + 16 * RT * w * D;
    const int64_t cell0 = (int64_t) blockIdx.x * kTileRows + 16 * RT * w;     // a split's rows, where there are several
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        sum[r] += __shfl_xor(sum[r], 16);
        sum[r] += __shfl_xor(sum[r], 32);
        const int x = 16 * r + i, row = row0 + 16 * RT * w + x;
        if (row < rows && k == 0) {
            if (parts) a.stat[cell0 + x] = make_float2(m[r], sum[r]);
            else if (a.rowq) keep_sum(a, hd * a.rows16 + row, m[r], sum[r]);
        }
        const float f = vref / kPScale * (parts ? 1.0f : inverse(sum[r]));
#pragma unroll
        for (int j = 0; j < NJ; ++j) *(f4 *) (mine + x * D + (((4 * j + k) ^ (x & (D / 4 - 1))) << 2)) = o[r][j] * f;
    }
    __syncthreads();
    auto rows_out = [&](auto store) {
#pragma unroll 4
        for (int u = 0; u < RT * D / 32; ++u) {
            const int at = 64 * u + l, x = at / (D / 8), d0 = at % (D / 8) * 8, row = row0 + 16 * RT * w + x;
            if (row >= rows) break;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f4 z = *(const f4 *) (mine + x * D + (((d0 + e) / 4 ^ (x & (D / 4 - 1))) << 2));
#pragma unroll
                for (int b = 0; b < 4; ++b) y[e + b] = z[b];
            }
            store(x, row, d0, y);
        }
    };
    if (parts)
        rows_out([&](int x, int, int d0, const float (&y)[8]) { store8<kF32>(a.part, (cell0 + x) * D + d0, true, y); });
    else
        by_type(a.o_type, [&](auto ot) {
            rows_out([&](int, int row, int d0, const float (&y)[8]) {
                store8<decltype(ot)::value>(a.o, s * a.os + row_at(a, row, g, a.orow, a.oh) + d0, a.ovec, y);
            });
        });
}

// acc of 64 slots: their probabilities of all rows, from rows in fp16 and the rows' sums that the attention kernels
// left.  Scores as there, bit for bit (the same order of dims: `lo` 8 of k_attend_few, 32 of k_attend_tile), so that
// none is above its row's maximum; K in registers, the next 16 rows on their way while these are worked on; the sum
// over rows is one over lanes i, then over them by way of LDS, in a fixed order.  A second pass over K rather than kept
// scores, which from 9 rows on are as many bytes as the keys and values.  Bound by issue (an exponential and four more
// instructions a score, at 3 waves a SIMD): 3 x 209 rows over 4,001 to 12,011 slots 35 us; 55 with rows in their own
// order, whose operands are halves of 16 lines a load, and lanes' sums by exchanges; 128 slots a wave need half the
// row reads, but leave one wave a SIMD (100 where this took 55), 4 waves a SIMD spill (82).
// grid (slot tiles / 4 * by, kv heads, sequences): `by` (1, 2 or 4) waves take the row tiles of one slot tile in turn
// and add up in their order.
template <int D>
__global__ __launch_bounds__(256) void k_attend_drawn(AttendArgs a, int by, int lo) {
    constexpr int NC = D / 32, NB = 4;
    __shared__ float part[4][64], sums[4][16][68];
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, i = l & 15, k = l >> 4;
    const int heads = a.c.n_kv_head, g = blockIdx.y, s = blockIdx.z;
    const int len = seq_len(a, s), n = seq_rows(a, s), rows = n * a.group;
    const int j0 = (blockIdx.x * (4 / by) + w / by) * 64;
    const int64_t hd = (int64_t) s * heads + g;
    float add[NB][4] = {};
    if (j0 < len && n) {
        const int last = len - 1;
        h8v kf[NB][NC];
        float ks[NB];
        const int off = lo == 8 ? 16 * k : 8 * k;
        const int8_t * kb = a.c.k + s * a.c.seq + g * a.c.head + off;
        const float * sb = a.c.ks + s * a.c.scale_seq + g * a.c.scale_head;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int8_t * p = kb + (int64_t) min(j0 + 16 * b + i, last) * D;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const u2 x = *(const u2 *) (p + lo * (c & 1) + 64 * (c >> 1));
                kf[b][c] = halves8(x[0], x[1]);
            }
            ks[b] = sb[min(j0 + 16 * b, last) / kBlk];
        }
        // the first row that sees slot j0
        const int rt0 = (a.causal ? max(j0 - (len - n), 0) * a.group / 16 : 0) + w % by, rt1 = (rows + 15) / 16;
        // from this row on a row sees all of these slots: none is masked (a row past the last one has the factor 0)
        const int clear = a.causal ? max(j0 + 63 - (len - n), 0) * a.group : 0;
        const uint16_t * qb = a.qh + hd * a.rows16 * D + 8 * l;
        const f4 * rb = a.rowq + hd * a.rows16 + i;
        h8v q[NC];
        f4 rq;
        auto fetch = [&](int rt) {
            rt = min(rt, rt1 - 1) * 16;
#pragma unroll
            for (int c = 0; c < NC; ++c) q[c] = *(const h8v *) (qb + (uint32_t) (rt * D + 512 * c));
            rq = rb[rt];
        };
        if (rt0 < rt1) fetch(rt0);
        for (int rt = rt0; rt < rt1; rt += by) {
            const int row = 16 * rt + i;
            f4 sc[NB];
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int b = 0; b < NB; ++b) sc[b] = mfma32(kf[b][c], q[c], c ? sc[b] : (f4){0.f, 0.f, 0.f, 0.f});
            const float factor = rq[0], top = rq[1], inv = rq[2];
            fetch(rt + by);
            if (16 * rt < clear) {
                const int lim = row_limit(a, len, n, token_of(a, min(row, rows - 1)));
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = __builtin_amdgcn_exp2f(sc[b][e] * (ks[b] * factor) - top);
                        add[b][e] = j0 + 16 * b + 4 * k + e < lim ? fmaf(x, inv, add[b][e]) : add[b][e];
                    }
                continue;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float f = ks[b] * factor;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    add[b][e] = fmaf(__builtin_amdgcn_exp2f(sc[b][e] * f - top), inv, add[b][e]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) *(f4 *) &sums[w][i][16 * b + 4 * k] = (f4){add[b][0], add[b][1], add[b][2], add[b][3]};
    __syncthreads();
    float own = 0.0f;
#pragma unroll
    for (int x = 0; x < 16; ++x) own += sums[w][x][l];
    part[w][l] = own;
    __syncthreads();
    const int j = j0 + l;
    if (w % by || !n || j >= len) return;
    float sum = part[w][l];
    for (int y = 1; y < by; ++y) sum += part[w + y][l];
    a.c.acc[s * a.c.acc_seq + g * a.c.acc_head + j] += sum;
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
    q3t_kv8 f, t;
    const int32_t * lens;
    int32_t len0, keep, sink, recent;
    int32_t * kept, * len_out;
};

constexpr int kEvT = 1024;

__device__ __forceinline__ int evict_len(const EvictArgs & a, int s) {
    const int64_t n = (int64_t) (a.lens ? a.lens[s] : 0) + a.len0;
    return (int) min(max(n, (int64_t) 0), (int64_t) a.f.n_slots);
}

// An fp32 weight as an integer of the same order; -0 as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictLds {
    uint32_t hist[256 * 8], total[256], cell[32 * kEvT / 64], sums[kEvT / 64], pick[3];   // hist: a copy for each lane mod 8
};

// The kept slots of one head with more than `keep` of them.  The threshold (the want-th largest weight of the slots
// between sink and recent) is found a byte at a time from the top by counting, until all slots that begin with its bytes
// are kept; then the kept slots are numbered in slot order, of those at the threshold the first ones: counts of 64 slots
// each by ballots, one prefix sum over them, and the place of each slot by the lanes before it.  R slots a thread at a
// time (slot base + 1,024 r + thread), as few as take them all, so that weights are read once: 2 x 8 heads of 600 slots
// 7.3 us (8.7 with 4), one of 2,049 8.5, 4 x 8 of 8,000 13 (25 with 32), 16 x 8 of 12,000 18 (31 with 32), 16 x 8 of 9,000
// to 32,768 41 (95 with weights read each time and numbered 1,024 at a time).  Bound by one workgroup's chain of counts.
template <int R>
__device__ __forceinline__ void select_slots(const EvictArgs & a, EvictLds & z, const float * acc, int len, int32_t * kept) {
    constexpr int kAt = R * kEvT;
    const int t = threadIdx.x, w = t >> 6, l = t & 63;
    const int lo = a.sink, hi = len - a.recent;     // len > keep >= sink + recent
    const bool once = len <= kAt;
    uint32_t key[R];
    auto read = [&](int base) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = base + kEvT * r + t;
            key[r] = i >= lo && i < hi ? order_of(acc[i]) : 0u;
        }
    };
    if (once) read(0);
    const bool some = a.keep > a.sink + a.recent;   // else sink and recent slots are all
    uint32_t want = (uint32_t) (a.keep - a.sink - a.recent), prefix = 0, mask = 0;
    for (int shift = some ? 24 : -8; shift >= 0; shift -= 8) {
        for (int i = t; i < 256 * 8; i += kEvT) z.hist[i] = 0;
        __syncthreads();
        for (int base = 0; base < len; base += kAt) {
            if (!once) read(base);
#pragma unroll
            for (int r = 0; r < R; ++r)             // key 0: no slot between sink and recent (no weight's is 0)
                if (key[r] && (key[r] & mask) == prefix) atomicAdd(&z.hist[(key[r] >> shift & 255) * 8 + (l & 7)], 1u);
        }
        __syncthreads();
        if (t < 256) {
            uint32_t n = 0;
#pragma unroll
            for (int x = 0; x < 8; ++x) n += z.hist[8 * t + x];
            z.total[t] = n;
        }
        __syncthreads();
        if (t < 64) {                               // the bin that the want-th largest is in, and how many are above it
            uint32_t c[4], above = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) c[x] = z.total[255 - 4 * l - x];
            uint32_t in = c[0] + c[1] + c[2] + c[3];
            const uint32_t own = in;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t y = __shfl_up(in, m);
                if (l >= m) in += y;
            }
            above = in - own;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (above < want && above + c[x] >= want) {
                    z.pick[0] = 255 - 4 * l - x;
                    z.pick[1] = above;
                    z.pick[2] = c[x];
                }
                above += c[x];
            }
        }
        __syncthreads();
        prefix |= z.pick[0] << shift;
        want -= z.pick[1];
        mask |= 255u << shift;
        const bool done = want == z.pick[2];        // all with these bytes are kept
        __syncthreads();
        if (done) break;
    }
    // prefix: the threshold, in the bytes of mask (those kept whole end in ones); want: how many slots at it are kept
    const uint32_t least = some ? max(prefix, 1u) : 0xffffffffu, most = some ? prefix | ~mask : 0xffffffffu;
    uint32_t over = 0, at = 0;                      // kept for sure, and at the threshold, so far
    for (int base = 0; base < len; base += kAt) {
        if (!once) read(base);
        auto sure = [&](int r) {
            const int i = base + kEvT * r + t;
            return key[r] ? key[r] > most : i < len;
        };
        auto tie = [&](int r) { return key[r] >= least && key[r] <= most; };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint64_t s = __ballot(sure(r)), e = __ballot(tie(r));
            if (l == 0) z.cell[r * (kEvT / 64) + w] = (uint32_t) __popcll(s) << 16 | (uint32_t) __popcll(e);
        }
        __syncthreads();
        const uint32_t own = t < R * (kEvT / 64) ? z.cell[t] : 0u;
        uint32_t in = own;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t y = __shfl_up(in, m);
            if (l >= m) in += y;
        }
        if (l == 63) z.sums[w] = in;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int x = 0; x < kEvT / 64; ++x) {
            const uint32_t y = z.sums[x];
            if (x < w) before += y;
            all += y;
        }
        if (t < R * (kEvT / 64)) z.cell[t] = in + before - own;
        __syncthreads();
        auto lanes_before = [](uint64_t m) {
            return __builtin_amdgcn_mbcnt_hi((uint32_t) (m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) m, 0u));
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool is = sure(r), ie = tie(r);
            const uint32_t c = z.cell[r * (kEvT / 64) + w];
            const uint32_t o = over + (c >> 16) + lanes_before(__ballot(is)), e = at + (c & 0xffffu) + lanes_before(__ballot(ie));
            if (is || (ie && e < want)) kept[o + min(e, want)] = base + kEvT * r + t;
        }
        over += all >> 16;
        at += all & 0xffffu;
        __syncthreads();
    }
}

// grid (kv heads, sequences): the kept slots of one head.
__global__ __launch_bounds__(kEvT) void k_evict_select(EvictArgs a) {
    __shared__ EvictLds z;
    const int t = threadIdx.x, h = blockIdx.x, s = blockIdx.y;
    const int len = evict_len(a, s), left = min(len, a.keep);
    int32_t * kept = a.kept + ((int64_t) s * a.f.n_kv_head + h) * a.keep;
    for (int i = left + t; i < a.keep; i += kEvT) kept[i] = -1;
    if (len <= a.keep) {
        for (int i = t; i < left; i += kEvT) kept[i] = i;
        return;
    }
    const float * acc = a.f.acc + s * a.f.acc_seq + h * a.f.acc_head;
    if (len <= kEvT) select_slots<1>(a, z, acc, len, kept);
    else if (len <= 4 * kEvT) select_slots<4>(a, z, acc, len, kept);
    else if (len <= 8 * kEvT) select_slots<8>(a, z, acc, len, kept);
    else if (len <= 16 * kEvT) select_slots<16>(a, z, acc, len, kept);
    else select_slots<32>(a, z, acc, len, kept);
}

constexpr int kMove = 64;                           // kept slots a workgroup of k_evict_move

// grid (kept slots / 64, kv heads, sequences).  One wave looks up the slots' old places and scales, and the new
// scales (the largest of each 16); then the codes, 16 bytes a thread at a time, all of a thread's on their way at
// once.  Bound by memory: 16 x 8 heads of 12,001 slots (790 MB) 158 us, 5.0 TB/s; a workgroup a block of 16, each
// thread looking up its own scales, took 431.
template <int D>
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
    constexpr int CH = D / 16, N = 2 * kMove * CH / 256;    // 16-byte pieces of a row; pieces a thread
    __shared__ int32_t from[kMove];
    __shared__ float ratio[2][kMove];
    const int t = threadIdx.x, h = blockIdx.y, s = blockIdx.z, at = blockIdx.x * kMove;
    const int32_t * kept = a.kept + ((int64_t) s * a.f.n_kv_head + h) * a.keep;
    const int64_t fsc = s * a.f.scale_seq + h * a.f.scale_head, tsc = s * a.t.scale_seq + h * a.t.scale_head;
    // here, where every head's selection has read the old lengths: len_out may be lens
    if (t == 0 && h == 0 && blockIdx.x == 0 && a.len_out) a.len_out[s] = min(evict_len(a, s), a.keep);
    if (t < kMove) {
        const int slot = at + t, f = slot < a.keep ? kept[slot] : -1;
        from[t] = f;
        float s0[2] = {0.0f, 0.0f};
        if (f >= 0) {
            s0[0] = a.f.ks[fsc + f / kBlk];
            s0[1] = a.f.vs[fsc + f / kBlk];
            a.t.acc[s * a.t.acc_seq + h * a.t.acc_head + slot] = a.f.acc[s * a.f.acc_seq + h * a.f.acc_head + f];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float s1 = s0[x];
#pragma unroll
            for (int m = 1; m < kBlk; m <<= 1) s1 = fmaxf(s1, __shfl_xor(s1, m));
            ratio[x][t] = s0[x] < s1 ? s0[x] / s1 : 1.0f;
            if (t % kBlk == 0 && f >= 0) (x ? a.t.vs : a.t.ks)[tsc + slot / kBlk] = s1;
        }
    }
    __syncthreads();
    u4 c[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int p = x * 256 + t, row = p / CH % kMove, f = from[row];
        const int8_t * src = (p / CH / kMove ? a.f.v : a.f.k) + s * a.f.seq + h * a.f.head + 16 * (p % CH);
        if (f >= 0) c[x] = *(const u4 *) (src + (int64_t) f * D);
    }
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int p = x * 256 + t, row = p / CH % kMove, is_v = p / CH / kMove;
        if (from[row] < 0) continue;
        const float r = ratio[is_v][row];
        if (r != 1.0f) {
            const u2 lo = rescale8((u2){c[x][0], c[x][1]}, r), hi = rescale8((u2){c[x][2], c[x][3]}, r);
            c[x] = (u4){lo[0], lo[1], hi[0], hi[1]};
        }
        *(u4 *) ((is_v ? a.t.v : a.t.k) + s * a.t.seq + h * a.t.head + (int64_t) (at + row) * D + 16 * (p % CH)) = c[x];
    }
}

// -------------------------------------------------------------------- read
struct ReadArgs {
    q3t_kv8 c;
    const int32_t * start;
    int32_t start0, n_rows, type;
    void * k, * v;
};

// grid (values / 8 / 256 of one sequence and of K or V, K or V, sequences): 8 values a thread.  Bound by memory: 1.18
// GB (the 16 x 8 heads above, to fp16) 225 us, 5.2 TB/s.
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
