// q3t_kv8.hip -- C ABI of the 8-bit attention cache's operators
// (include/q3t_kv8.h): argument checks, launch shapes and workspaces.

#include "q3t_kv8_kernels.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <string>

using namespace q3t;

namespace {

thread_local char t_err[256] = "";

int refuse(const char * what) {
    snprintf(t_err, sizeof t_err, "%s", what);
    return -1;
}

// `device` made current for the length of a call.
struct OnDevice {
    int was = -1, dev;
    bool ok = true;
    explicit OnDevice(int d) : dev(d) {
        if (hipGetDevice(&was) != hipSuccess || was < 0) ok = false;
        else if (was != d && hipSetDevice(d) != hipSuccess) ok = false;
    }
    ~OnDevice() { if (ok && was != dev) (void) hipSetDevice(was); }
};

int launched(const char * what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    snprintf(t_err, sizeof t_err, "%s: %s", what, hipGetErrorString(e));
    return -2;
}

#define ON_DEVICE(d)                                              \
    OnDevice on_(d);                                              \
    if (!on_.ok) {                                                \
        (void) hipGetLastError();                                 \
        return refuse("no such HIP device");                      \
    }

bool is16(const void * p) { return ((uintptr_t) p & 15) == 0; }
bool type_ok(int t) { return t == kv8::kF32 || t == kv8::kF16 || t == kv8::kBF16; }
int type_size(int t) { return t == kv8::kF32 ? 4 : 2; }
bool strides16(int type, std::initializer_list<int64_t> s) {
    for (int64_t x : s) if (x * type_size(type) % 16) return false;
    return true;
}

int check_cache(const q3t_kv8 * c, bool acc) {
    if (!c) return refuse("null cache");
    if (!c->k || !c->v || !c->ks || !c->vs) return refuse("null cache pointer");
    if (acc && !c->acc) return refuse("the cache keeps no weights (acc is null)");
    if (c->head_dim != 64 && c->head_dim != 128) return refuse("head_dim must be 64 or 128");
    if (c->n_seq < 1 || c->n_seq > 65535) return refuse("n_seq must be 1 to 65535");
    if (c->n_kv_head < 1 || c->n_kv_head > 4096) return refuse("n_kv_head must be 1 to 4096");
    // a grid's threads along one axis are counted in 32 bits: here, and in the bounds on rows and tokens below
    if ((int64_t) c->n_seq * c->n_kv_head > 1 << 23) return refuse("n_seq * n_kv_head must be at most 2^23");
    if (c->n_slots < 16 || c->n_slots % 16 || c->n_slots > 1 << 29) return refuse("n_slots must be a multiple of 16, 16 to 2^29");
    if (!is16(c->k) || !is16(c->v) || c->seq % 16 || c->head % 16) return refuse("codes must be 16-byte aligned");
    return 0;
}

}  // namespace

extern "C" {

const char * q3t_kv8_last_error(void) { return t_err; }

int q3t_kv8_rope_freqs(int32_t rot_dim, double theta, int32_t scaling, double factor, int32_t n_trained,
                       double * freq_out) {
    t_err[0] = 0;
    if (!freq_out) return refuse("null frequencies");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 256) return refuse("rot_dim must be even, 2 to 256");
    if (!(theta > 0.0) || !std::isfinite(theta)) return refuse("theta must be positive");
    if (scaling < 0 || scaling > 3) return refuse("unknown scaling");
    if (scaling && (!(factor >= 1.0) || !std::isfinite(factor))) return refuse("factor must be at least 1");
    if (scaling == 2 && rot_dim == 2) return refuse("this scaling needs rot_dim > 2");
    if (scaling == 3 && n_trained < 1) return refuse("this scaling needs n_trained");
    if (scaling == 2) theta *= std::pow(factor, rot_dim / (rot_dim - 2.0));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / rot_dim);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double turns = n_trained * f / (2.0 * M_PI);
            const double keep = std::min(std::max(std::log(turns) / std::log(32.0), 0.0), 1.0);
            f = f * keep + f / factor * (1.0 - keep);
        }
        freq_out[i] = f;
    }
    return 0;
}

int q3t_kv8_rope(int32_t device, const q3t_kv8_rope_rows * rows, int32_t n, int64_t n_tokens, int32_t head_dim,
                 int32_t rot_dim, int32_t interleaved, const int32_t * pos, int32_t pos0, const double * freq,
                 float mscale, float eps, void * stream) {
    t_err[0] = 0;
    if (!rows || !freq) return refuse("null argument");
    if (n < 1 || n > 4) return refuse("1 to 4 tensors a call");
    if (n_tokens < 0 || n_tokens > 1 << 26) return refuse("n_tokens must be 0 to 2^26");
    if (head_dim < 16 || head_dim % 16 || head_dim > 256) return refuse("head_dim must be a multiple of 16, up to 256");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim) return refuse("rot_dim must be even, 2 to head_dim");
    kv8::RopeArgs a{};
    for (int i = 0; i < n; ++i) {
        const q3t_kv8_rope_rows & r = rows[i];
        if (n_tokens && (!r.x || !r.y)) return refuse("null rows");
        if (!type_ok(r.x_type) || !type_ok(r.y_type)) return refuse("types must be F32, F16 or BF16");
        if (r.n_head < 1 || r.n_head > 65535) return refuse("n_head must be 1 to 65535");
        if (r.x == r.y && (r.x_type != r.y_type || r.x_token != r.y_token || r.x_head != r.y_head))
            return refuse("in place needs the same type and strides");
        a.r[i] = kv8::RopeRows{r.x, r.y, r.x_token, r.x_head, r.y_token, r.y_head, r.gain, r.n_head, r.x_type, r.y_type,
                               is16(r.x) && is16(r.y) && strides16(r.x_type, {r.x_token, r.x_head}) &&
                                   strides16(r.y_type, {r.y_token, r.y_head})};
    }
    if (!n_tokens) return 0;
    ON_DEVICE(device);
    a.pos = pos; a.pos0 = pos0; a.freq = freq; a.n_tokens = n_tokens; a.head_dim = head_dim; a.rot = rot_dim;
    a.inter = interleaved != 0; a.mscale = mscale; a.eps = eps;
    // up to 8 tokens a workgroup, while there are two workgroups a CU
    a.n = n;
    a.per = (int) std::min<int64_t>(std::max<int64_t>(n_tokens / 512, 1), kv8::kRopeTok);
    hipLaunchKernelGGL(kv8::k_rope, dim3((unsigned) ((n_tokens + a.per - 1) / a.per)), dim3(kv8::kRopeT), 0, (hipStream_t) stream, a);
    return launched("rope");
}

int q3t_kv8_append(int32_t device, const q3t_kv8 * c, const void * k, const void * v, int32_t type, int64_t x_seq,
                   int64_t x_row, int64_t x_head, int32_t n_rows, const int32_t * start, int32_t start0,
                   const int32_t * n_new, void * stream) {
    t_err[0] = 0;
    if (check_cache(c, false)) return -1;
    if (n_rows < 0 || n_rows > 1 << 26) return refuse("n_rows must be 0 to 2^26");
    if (!n_rows) return 0;
    if (!k || !v) return refuse("null rows");
    if (!type_ok(type)) return refuse("type must be F32, F16 or BF16");
    ON_DEVICE(device);
    kv8::AppendArgs a{*c, k, v, x_seq, x_row, x_head, start, n_new, start0, n_rows, type,
                      is16(k) && is16(v) && strides16(type, {x_seq, x_row, x_head})};
    // rows that begin at a block's last slot touch the most blocks
    const dim3 grid((unsigned) (((int64_t) n_rows + 2 * kv8::kBlk - 2) / kv8::kBlk), 2 * c->n_kv_head, c->n_seq);
    auto go = [&](auto d, auto t) {
        hipLaunchKernelGGL((kv8::k_append<decltype(d)::value, decltype(t)::value>), grid, dim3(2 * decltype(d)::value), 0,
                           (hipStream_t) stream, a);
    };
    auto go_t = [&](auto d) {
        if (type == kv8::kF32) go(d, std::integral_constant<int, kv8::kF32>{});
        else if (type == kv8::kF16) go(d, std::integral_constant<int, kv8::kF16>{});
        else go(d, std::integral_constant<int, kv8::kBF16>{});
    };
    if (c->head_dim == 64) go_t(std::integral_constant<int, 64>{});
    else go_t(std::integral_constant<int, 128>{});
    return launched("append");
}

static int check_attend(const q3t_kv8 * c, const q3t_kv8_attend_args * a) {
    if (!a) return refuse("null arguments");
    if (check_cache(c, a->weights != 0)) return -1;
    if (a->q_type != kv8::kF16 && a->q_type != kv8::kBF16) return refuse("q must be F16 or BF16");
    if (!type_ok(a->o_type)) return refuse("out must be F32, F16 or BF16");
    if (a->n_rows < 0 || a->n_rows > 65535) return refuse("n_rows must be 0 to 65535");
    if (a->n_head < 1 || a->n_head % c->n_kv_head || a->n_head / c->n_kv_head > 32 || a->n_head > 65535)
        return refuse("n_head must be a multiple of n_kv_head, at most 32 times as many");
    if (a->max_len < 0 || a->max_len > c->n_slots) return refuse("max_len must be 0 to n_slots");
    if (!(a->scale == a->scale) || std::isinf(a->scale)) return refuse("scale must be finite");
    return 0;
}

}  // extern "C"

namespace {

// How a call runs: its kernels, splits and the parts of its workspace (bytes).
struct AttendPlan {
    bool few, whole, scored, drawn;
    int rt, row_tiles, units, split_tiles, n_split, score_len, rows16;
    int64_t part, stat, split, score, qh, rowq, total;
};

AttendPlan plan_attend(const q3t_kv8 * c, const q3t_kv8_attend_args * a) {
    AttendPlan p{};
    const int64_t len = a->max_len ? a->max_len : c->n_slots, heads = (int64_t) c->n_seq * c->n_kv_head;
    const int64_t group = a->n_head / c->n_kv_head, rows = a->n_rows * group, tiles = (len + 63) / 64;
    p.few = rows <= 32;
    int64_t st;
    if (p.few) {
        p.rt = rows <= 16 ? 1 : 2;
        // short contexts in one workgroup a head, without a join (one row of 8 x 2 heads with weights over 64, 250, 512,
        // 1,000 slots: 7.4, 8.3, 10.2, 13.7 us; split and joined 10.8, 12.0, 11.2, 11.4)
        p.whole = tiles <= kv8::kWhole;
        // 4 tiles (one a wave) to 16 a split, so that there are about 1,024 workgroups: four a CU
        st = (std::min<int64_t>(std::max<int64_t>((heads * tiles + 1023) / 1024, 4), 16) + 3) & ~(int64_t) 3;
    } else {
        // As many workgroups as run at once, two a CU, or splits of 4 tiles if those are fewer (of 8, 6, 4, 3, 2 tiles: 4 x
        // 16 rows of one kv head over 7,207 and 21,659 slots, all kernels, 33, 31, 29, 29, 30 us; 64 x 2 of 8 over 2,000 34,
        // 32, 31, 28, 27; 1,000 x 2 of 8 over their own 50, 48, 51, 51, 53): more start a second turn
        // (512, 640, 768, 1,024: 3 x 209 rows over 4,001 to 12,011 slots 84, 92, 85, 91 us, 2,049 rows over their own
        // 49, 56, 57, 57).
        p.row_tiles = (int) ((rows + kv8::kTileRows - 1) / kv8::kTileRows);
        const int64_t whole = heads * p.row_tiles;
        p.units = whole < kv8::kUnits ? (int) std::min<int64_t>(kv8::kUnits, whole * ((tiles + kv8::kLeast - 1) / kv8::kLeast)) : 0;
        if (p.units == whole) p.units = 0;
        st = tiles;
    }
    if (p.whole) st = tiles;
    else if (p.few) st = std::max(st, (tiles + kv8::kSplitMax - 1) / kv8::kSplitMax);
    p.scored = a->weights && rows <= 8 && !p.whole;
    p.drawn = a->weights && rows > 8;
    p.split_tiles = (int) st;
    p.n_split = (int) ((tiles + st - 1) / st);
    p.score_len = (int) (tiles * 64);
    p.rows16 = (int) ((rows + 15) / 16 * 16);
    auto take = [&](int64_t bytes) { const int64_t at = p.total; p.total += (bytes + 255) / 256 * 256; return at; };
    const int64_t cells = p.units ? (int64_t) p.units * kv8::kTileRows : heads * p.n_split * rows;
    if (p.units || p.n_split > 1) p.part = take(cells * c->head_dim * 4);
    if (p.units || p.n_split > 1 || p.scored) p.stat = take(cells * 8);
    if (p.units) p.split = take(heads * p.row_tiles * 8);
    if (p.scored) p.score = take(heads * rows * p.score_len * 4);
    if (p.drawn) p.qh = take(heads * p.rows16 * c->head_dim * 2);
    if (p.drawn) p.rowq = take(heads * p.rows16 * 16);
    return p;
}

template <int D>
void launch_attend(kv8::AttendArgs a, const AttendPlan & p, hipStream_t st) {
    const int rows = a.n_rows * a.group, H = a.c.n_kv_head, S = a.c.n_seq;
    if (p.few) {
        const dim3 grid(H, p.n_split, S);
        if (p.whole && p.rt == 1) hipLaunchKernelGGL((kv8::k_attend_few<D, 1, 8>), grid, dim3(512), 0, st, a);
        else if (p.whole) hipLaunchKernelGGL((kv8::k_attend_few<D, 2, 8>), grid, dim3(512), 0, st, a);
        else if (p.rt == 1) hipLaunchKernelGGL((kv8::k_attend_few<D, 1, 4>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((kv8::k_attend_few<D, 2, 4>), grid, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL(kv8::k_attend_tile<D>, p.units ? dim3(p.units) : dim3(H * S, p.row_tiles), dim3(kv8::kTileT), 0, st, a);
    }
    // a workgroup a row from 17 splits on (209 x 2 rows of 8 heads in 16 splits: 9.9 us so, 6.5 as a row of several; 32 x 8 of
    // 4 in 64 splits 6.3, 7.2)
    const bool many = p.few ? p.n_split > 16 : p.units > (int64_t) 16 * H * S * p.row_tiles;
    a.row_blocks = p.n_split == 1 && !p.units ? 0 : many ? rows : (rows + 1024 / D - 1) / (1024 / D);
    const dim3 join(a.row_blocks + (p.scored ? (a.max_len + 1023) / 1024 : 0), H, S);
    if (join.x && many) hipLaunchKernelGGL((kv8::k_attend_join<D, true>), join, dim3(256), 0, st, a);
    else if (join.x) hipLaunchKernelGGL((kv8::k_attend_join<D, false>), join, dim3(256), 0, st, a);
    if (p.drawn) {
        // waves that share a slot tile, where one a tile would leave CUs without work (each loads the tile's keys; 1, 2
        // and 4 waves: 3 x 209 rows over 4,001 to 12,011 slots, 1,128 workgroups of one a tile, 37, 43, 57 us; over 12,011
        // of one sequence, 376, 23, 21, 28; 2,049 rows over their own, 66, 118, 63, 37)
        const int64_t tiles = (a.max_len + 63) / 64, groups = tiles * H * S / 4;
        const int by = rows <= 48 || groups >= 512 ? 1 : groups >= 256 ? 2 : 4;
        hipLaunchKernelGGL(kv8::k_attend_drawn<D>, dim3((unsigned) ((tiles * by + 3) / 4), H, S), dim3(256), 0, st, a, by,
                           p.few ? 8 : 32);
    }
}

}  // namespace

extern "C" {

int64_t q3t_kv8_attend_ws(const q3t_kv8 * c, const q3t_kv8_attend_args * a) {
    t_err[0] = 0;
    if (check_attend(c, a)) return -1;
    return plan_attend(c, a).total;
}

int q3t_kv8_attend(int32_t device, const q3t_kv8 * c, const q3t_kv8_attend_args * p, void * ws, int64_t ws_bytes,
                   void * stream) {
    t_err[0] = 0;
    if (check_attend(c, p)) return -1;
    if (!p->n_rows) return 0;
    if (!p->q || !p->out) return refuse("null rows");
    const AttendPlan plan = plan_attend(c, p);
    if (plan.total > 0 && (!ws || ws_bytes < plan.total)) return refuse("workspace too small");
    if (!is16(ws)) return refuse("workspace must be 16-byte aligned");
    ON_DEVICE(device);
    kv8::AttendArgs a{};
    a.c = *c; a.q = p->q; a.o = p->out;
    a.qs = p->q_seq; a.qr = p->q_row; a.qhd = p->q_head; a.os = p->o_seq; a.orow = p->o_row; a.oh = p->o_head;
    a.lens = p->lens; a.n_new = p->n_new; a.len0 = p->len0; a.q_type = p->q_type; a.o_type = p->o_type;
    a.n_rows = p->n_rows; a.n_head = p->n_head; a.group = p->n_head / c->n_kv_head;
    a.max_len = p->max_len ? p->max_len : c->n_slots;
    a.per_group = 1.0f / a.group;
    a.causal = p->causal != 0; a.weights = p->weights != 0; a.scale = p->scale;
    a.qvec = is16(p->q) && strides16(p->q_type, {p->q_seq, p->q_row, p->q_head});
    a.ovec = is16(p->out) && strides16(p->o_type, {p->o_seq, p->o_row, p->o_head});
    a.split_tiles = plan.split_tiles; a.n_split = plan.n_split; a.row_tiles = plan.row_tiles;
    a.score_len = plan.score_len; a.rows16 = plan.rows16;
    char * w = (char *) ws;
    a.units = plan.units;
    a.most = (a.max_len + 63) / 64;
    if (plan.units || plan.n_split > 1) a.part = (float *) (w + plan.part);
    if (plan.units || plan.n_split > 1 || plan.scored) a.stat = (float2 *) (w + plan.stat);
    if (plan.units) a.split = (int2 *) (w + plan.split);
    if (plan.scored) a.score = (float *) (w + plan.score);
    if (plan.drawn) { a.qh = (uint16_t *) (w + plan.qh); a.rowq = (kv8::f4 *) (w + plan.rowq); }
    if (c->head_dim == 64) launch_attend<64>(a, plan, (hipStream_t) stream);
    else launch_attend<128>(a, plan, (hipStream_t) stream);
    return launched("attend");
}

int q3t_kv8_evict(int32_t device, const q3t_kv8 * from, const q3t_kv8 * to, const int32_t * lens, int32_t len0,
                  int32_t n_keep, int32_t n_sink, int32_t n_recent, int32_t * kept, int32_t * len_out, void * stream) {
    t_err[0] = 0;
    if (check_cache(from, true) || check_cache(to, true)) return -1;
    if (from->n_seq != to->n_seq || from->n_kv_head != to->n_kv_head || from->head_dim != to->head_dim)
        return refuse("the caches' sequences, heads and head_dim must be the same");
    if (from->k == to->k || from->v == to->v || from->ks == to->ks || from->vs == to->vs || from->acc == to->acc)
        return refuse("evict needs other memory to write to");
    if (n_keep < 1 || n_keep > to->n_slots) return refuse("n_keep must be 1 to the slots of `to`");
    if (n_sink < 0 || n_recent < 0 || (int64_t) n_sink + n_recent > n_keep)
        return refuse("n_sink + n_recent must be at most n_keep");
    if (!kept) return refuse("null kept");
    ON_DEVICE(device);
    kv8::EvictArgs a{*from, *to, lens, len0, n_keep, n_sink, n_recent, kept, len_out};
    hipLaunchKernelGGL(kv8::k_evict_select, dim3(from->n_kv_head, from->n_seq), dim3(kv8::kEvT), 0, (hipStream_t) stream, a);
    const dim3 grid((n_keep + kv8::kMove - 1) / kv8::kMove, from->n_kv_head, from->n_seq);
    if (from->head_dim == 64) hipLaunchKernelGGL(kv8::k_evict_move<64>, grid, dim3(256), 0, (hipStream_t) stream, a);
    else hipLaunchKernelGGL(kv8::k_evict_move<128>, grid, dim3(256), 0, (hipStream_t) stream, a);
    return launched("evict");
}

int q3t_kv8_read(int32_t device, const q3t_kv8 * c, const int32_t * start, int32_t start0, int32_t n_rows, int32_t type,
                 void * k, void * v, void * stream) {
    t_err[0] = 0;
    if (check_cache(c, false)) return -1;
    if (n_rows < 0 || (int64_t) n_rows * c->n_kv_head * c->head_dim >= (int64_t) 1 << 35)
        return refuse("n_rows must not be negative, nor n_rows * n_kv_head * head_dim 2^35");
    if (!type_ok(type)) return refuse("type must be F32, F16 or BF16");
    if (!is16(k) || !is16(v)) return refuse("outputs must be 16-byte aligned");
    if (!n_rows || (!k && !v)) return 0;
    ON_DEVICE(device);
    kv8::ReadArgs a{*c, start, start0, n_rows, type, k, v};
    const int64_t per = (int64_t) n_rows * c->n_kv_head * c->head_dim;
    const int64_t blocks = (per / 8 + 255) / 256;
    const dim3 grid((unsigned) blocks, 2, c->n_seq);
    auto go = [&](auto d, auto t) {
        hipLaunchKernelGGL((kv8::k_read<decltype(d)::value, decltype(t)::value>), grid, dim3(256), 0, (hipStream_t) stream, a);
    };
    auto go_t = [&](auto d) {
        if (type == kv8::kF32) go(d, std::integral_constant<int, kv8::kF32>{});
        else if (type == kv8::kF16) go(d, std::integral_constant<int, kv8::kF16>{});
        else go(d, std::integral_constant<int, kv8::kBF16>{});
    };
    if (c->head_dim == 64) go_t(std::integral_constant<int, 64>{});
    else go_t(std::integral_constant<int, 128>{});
    return launched("read");
}

}  // extern "C"
