"""The 8-bit cache's operators against their definitions in 64 bits, at the
sizes, masks, strides and values where they can go wrong, and together as a
session uses them.

u = 2^-24 is half a step of fp32 (relative).  Bounds count roundings; they are
stated where they are used.
"""
import math

import numpy as np
import pytest
import torch

from qwen3_tts_amd import kv8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}    # half the step of the type's smallest values
T16 = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, want, bound):
    """got (any float type) is within `bound` of want (64 bits), both finite there; NaN where want is NaN."""
    got = got.double()
    assert got.shape == want.shape
    nan = want.isnan()
    wrong = (got.isnan() != nan).sum().item()
    assert not wrong, f"{wrong} of {nan.numel()} values are NaN where they should not be, or the other way"
    bound = bound.expand_as(want) if torch.is_tensor(bound) else torch.full_like(want, bound)
    over = ((got - want).abs() - bound)[~nan]
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"off by up to {worst} more than the bound"


# ---------------------------------------------------------------- rotary
def rope64(x, pos, freq, gain, inter, mscale, eps):
    """(result, sum of the magnitudes of its two terms)"""
    z = x.double()
    if gain is not None:
        z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    half = freq.numel()
    i = torch.arange(half, device=x.device)
    p, q = (2 * i, 2 * i + 1) if inter else (i, i + half)
    a = (pos.double()[:, None] * freq)[:, None]
    y, mag = z.clone(), z.abs()
    y[..., p] = (z[..., p] * a.cos() - z[..., q] * a.sin()) * mscale
    y[..., q] = (z[..., q] * a.cos() + z[..., p] * a.sin()) * mscale
    m = (z[..., p].abs() + z[..., q].abs()) * mscale
    mag[..., p], mag[..., q] = m, m
    return y, mag


def rope_bound(y, mag, t):
    # sines and cosines: the angle rounded to fp32 (2^-23 up to pi), the function (2^-22 at most), times mscale; then
    # two products and a sum; the norm: 16 squares a lane, 4 lane sums, root, division, two products (under 32 u).
    # Together under 48 u of the terms' magnitude; then one rounding to the output's type.
    return mag * 48 * U + (y.abs() + mag * 48 * U) * HALF[t] + TINY[t]


ROPE = [(1, [16, 8], 128, 128), (1, [1], 16, 2), (37, [16, 8], 128, 128), (7, [3], 128, 64), (19, [5, 1], 128, 6),
        (65, [2], 64, 64), (9, [4], 96, 96), (5, [7], 256, 256), (3, [33], 80, 34), (131, [32, 4], 64, 62)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("t,heads,d,rot", ROPE)
def test_rope(t, heads, d, rot, norm, inter):
    g = gen(t * 1000 + d + rot)
    freq = torch.from_numpy(kv8.rope_freqs(rot, 1e6, "turns", 4.0, 32768)).cuda()
    pos = torch.randint(-5, 40000, (t,), generator=g, device="cuda", dtype=torch.int32)
    types = [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
             (torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)]
    for ti, to in types:
        xs = [(3 * torch.randn(t, h, d, generator=g, device="cuda")).to(ti) for h in heads]
        gains = [1 + 0.2 * torch.randn(d, generator=g, device="cuda") if norm else None for _ in heads]
        ys = kv8.rope(xs, pos, freq, gains=gains, dtype=to, interleaved=inter, mscale=1.1, eps=1e-6)
        for x, gain, y in zip(xs, gains, ys):
            want, mag = rope64(x, pos, freq, gain, inter, 1.1, 1e-6)
            assert y.dtype == to
            within(y, want, rope_bound(want, mag, to))


def test_rope_far_positions():
    """Angles of 2^31 turns' worth: 64 bits carry pos * freq to 2^-22, far below what is asserted."""
    freq = torch.from_numpy(kv8.rope_freqs(128, 1e6)).cuda()
    pos = ints([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 1000003])
    x = torch.randn(6, 3, 128, generator=gen(1), device="cuda")
    y, = kv8.rope([x], pos, freq)
    want, mag = rope64(x, pos, freq, None, False, 1.0, 0)
    # two angles of up to 2^31 in 64 bits may differ by their own rounding, 2^-22 each
    within(y, want, rope_bound(want, mag, torch.float32) + mag * 2.0 ** -21)


@pytest.mark.parametrize("inter", [False, True])
def test_rope_strides_and_in_place(inter):
    g = gen(2)
    freq = torch.from_numpy(kv8.rope_freqs(96, 1e4)).cuda()
    pos = torch.arange(11, device="cuda", dtype=torch.int32) * 77
    # q and k inside fused rows of 129 values more (odd strides: not 16-byte aligned), and heads before tokens
    fused = torch.randn(11, 6 * 128 + 129, generator=g, device="cuda").half()
    before = fused.clone()
    q = fused[:, :512].view(11, 4, 128) if fused[:, :512].is_contiguous() else fused[:, :512].unflatten(1, (4, 128))
    k = fused[:, 513:513 + 256].unflatten(1, (2, 128))
    wants = [rope64(v, pos, freq, None, inter, 1.0, 0) for v in (q, k)]
    kv8.rope([q, k], pos, freq, outs=[q, k], interleaved=inter)
    for v, (w, m) in zip((q, k), wants):
        within(v, w, rope_bound(w, m, torch.float16))
    rest = torch.ones(fused.shape[1], dtype=torch.bool, device="cuda")
    rest[:512] = False
    rest[513:769] = False
    assert torch.equal(fused[:, rest], before[:, rest])
    x = torch.randn(5, 11, 128, generator=g, device="cuda").transpose(0, 1)
    out = torch.zeros(5, 11, 128, device="cuda").transpose(0, 1)
    kv8.rope([x], pos, freq, outs=[out], interleaved=inter)
    w, m = rope64(x, pos, freq, None, inter, 1.0, 0)
    within(out, w, rope_bound(w, m, torch.float32))


def test_rope_position_sums_past_32_bits():
    """pos + pos0 beyond an int32."""
    x = torch.randn(4, 2, 64, generator=gen(14), device="cuda")
    pos, freq = ints([2 ** 31 - 1, 2 ** 31 - 50, 0, 7]), torch.from_numpy(kv8.rope_freqs(64, 1e6)).cuda()
    y, pos0 = torch.empty_like(x), 2 ** 31 - 1
    rows = kv8._pack_rope(x.data_ptr(), y.data_ptr(), 128, 64, 128, 64, 0, 2, 0, 0)
    kv8._check(kv8.load_kv8_library().q3t_kv8_rope(x.get_device(), rows, 1, 4, 64, 64, 0, pos.data_ptr(), pos0, freq.data_ptr(),
                                                   1.0, 0.0, kv8._stream(x.get_device())), "rope")
    want, mag = rope64(x, pos.long() + pos0, freq, None, False, 1.0, 0.0)
    within(y, want, rope_bound(want, mag, torch.float32))


def test_rope_nothing_and_refusals():
    freq = torch.from_numpy(kv8.rope_freqs(64, 1e4)).cuda()
    y, = kv8.rope([torch.empty(0, 4, 64, device="cuda")], ints([]), freq)
    assert y.shape == (0, 4, 64)
    x = torch.randn(3, 4, 64, device="cuda")
    for bad in [dict(pos=ints([1, 2])), dict(pos=torch.zeros(3, device="cuda")), dict(freq=freq.float()), dict(freq=freq.cpu()),
                dict(freq=torch.cat([freq, freq])), dict(xs=[x.double()]), dict(xs=[x, x[:2]]), dict(xs=[x.transpose(1, 2)]),
                dict(gains=[torch.ones(32, device="cuda")]), dict(outs=[x.half(), x])]:
        a = dict(xs=[x], pos=ints([1, 2, 3]), freq=freq) | bad
        with pytest.raises(kv8.Kv8Error):
            kv8.rope(a.pop("xs"), a.pop("pos"), a.pop("freq"), **a)


# ---------------------------------------------------------------- append
def snapshot(c):
    return [None if t is None else t.clone() for t in c.tensors]


def append64(c, k, v, start, n_new):
    """The cache after append by its definition: per block new scales and codes before rounding, as 64-bit values.
    Returns {name: (codes before rounding [S, H, C, D], scales [S, H, C / 16], stored [S, H, C])}."""
    out = {}
    for name, codes, scales, x in (("k", c.tensors[0], c.tensors[2], k), ("v", c.tensors[1], c.tensors[3], v)):
        q, s = codes.double().cpu(), scales.double().cpu()
        x = x.double().cpu()
        new = torch.zeros(q.shape[:3], dtype=torch.bool)
        slots = q.shape[2]
        for b in range(q.shape[0]):
            n = x.shape[1] if n_new is None else min(max(n_new[b], 0), x.shape[1])
            rows = [i for i in range(n) if 0 <= start[b] + i < slots]
            for blk in sorted({(start[b] + i) // 16 for i in rows}):
                mine = [i for i in rows if (start[b] + i) // 16 == blk]
                at = [start[b] + i for i in mine]
                for h in range(q.shape[1]):
                    y = x[b, mine, h]
                    a = torch.where(y.isfinite(), y.abs(), 0.0).max() / 127
                    begun = start[b] > blk * 16
                    s1 = max(s[b, h, blk].item(), a.item()) if begun else a.item()
                    if begun and s1 > s[b, h, blk]:
                        q[b, h, blk * 16:start[b]] *= s[b, h, blk] / s1
                    s[b, h, blk] = s1
                    y = y / s1 if s1 > 0 else torch.zeros_like(y)
                    q[b, h, at] = torch.where(y.isnan(), 0.0, y).clamp(-127, 127)
                    new[b, h, at] = True
        out[name] = (q.cuda(), s.cuda(), new.cuda())
    return out


def check_append(c, before, want, acc_before):
    for name, codes, scales in (("k", c.tensors[0], c.tensors[2]), ("v", c.tensors[1], c.tensors[3])):
        q, s, new = want[name]
        within(scales, s, s.abs() * U)
        # x / s: the scale's rounding and the division's, of up to 127; then to the nearest whole number
        within(codes.float(), q, 0.5 + 127 * 4 * U)
        assert torch.equal((codes.double() - q).abs() > 0.5 + 1e-4, torch.zeros_like(codes, dtype=torch.bool))
    if acc_before is not None:
        assert torch.equal(c.tensors[4], torch.where(want["k"][2], 0.0, acc_before))


APPEND = [(1, 1, 128, 1, [0], None), (1, 2, 128, 1, [15], None), (2, 3, 64, 5, [14, 16], None), (3, 2, 128, 40, [0, 7, 31], None),
          (3, 2, 64, 33, [1, 63, 95], [33, 0, 7]), (2, 1, 128, 17, [100, 127], [17, 40]), (2, 2, 128, 9, [-3, -20], None),
          (1, 1, 64, 200, [3], [-1]), (2, 2, 128, 6, [126, 128], None)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("s,h,d,n,start,n_new", APPEND)
def test_append(s, h, d, n, start, n_new, dtype):
    g = gen(s * 100 + n)
    c = kv8.empty(s, h, 128, d)
    kv8.append(c, *(torch.randn(s, 128, h, d, generator=g, device="cuda") for _ in range(2)), ints([0] * s))
    c.tensors[4].uniform_(0.1, 1.0, generator=g)
    before = snapshot(c)
    # rows that grow: the later blocks' scales differ, and a begun block's scale grows, stays or is far above
    for grow in (3.0, 0.01):
        acc = c.tensors[4].clone()
        k, v = (grow * torch.randn(s, n, h, d, generator=g, device="cuda").to(dtype) for _ in range(2))
        want = append64(c, k, v, start, n_new)
        kv8.append(c, k, v, ints(start), None if n_new is None else ints(n_new))
        check_append(c, before, want, acc)


def test_append_special_values():
    c = kv8.empty(1, 1, 64, 64)
    k = torch.randn(1, 20, 1, 64, generator=gen(3), device="cuda")
    k[0, 3] = math.nan
    k[0, 4, 0, :5] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0])
    k[0, 16:] = 0.0
    v = torch.full_like(k, math.inf)
    want = append64(c, k, v, [0], None)
    kv8.append(c, k, v, ints([0]))
    check_append(c, None, want, None)
    assert (c.tensors[0][0, 0, 3] == 0).all() and c.tensors[0][0, 0, 4, :3].tolist() == [127, -127, 0]
    assert c.tensors[2][0, 0, 1] == 0 and (c.tensors[1] == 0).all() and (c.tensors[3] == 0).all()
    # tiny and huge rows: scales near both ends of fp32
    for size in (1e-36, 1e36):
        k = size * torch.randn(1, 17, 1, 64, generator=gen(4), device="cuda")
        want = append64(c, k, k, [32], None)
        kv8.append(c, k, k, ints([32]))
        check_append(c, None, want, None)


def test_append_one_by_one_and_strided():
    """Rows one at a time: a value is off by half a step when stored and by half a step of the new scale at each growth of
    its block's scale."""
    g = gen(5)
    wide = torch.randn(2, 4, 21, 3 * 64 + 8, generator=g, device="cuda")      # heads before rows, odd offsets
    k, v = (wide[..., o:o + 64].transpose(1, 2) for o in (1, 65))
    c = kv8.empty(2, 4, 48, 64)
    for i in range(21):
        kv8.append(c, k[:, i:i + 1], v[:, i:i + 1], ints([9 + i, 3 + i]))
    for name, x, scale in (("k", k, c.tensors[2]), ("v", v, c.tensors[3])):
        got = kv8.read(c, ints([9, 3]), 21)["kv".index(name)]
        step = torch.stack([scale[b][:, (torch.arange(21, device="cuda") + [9, 3][b]) // 16].T for b in range(2)])
        # at most 15 growths, each adding half a step of a scale no larger than the last one
        within(got, x.double(), 8.1 * step.double()[..., None])
        # and as a rule far less: the scales of random rows grow a few times
        assert ((got - x).abs() / step[..., None]).mean() < 0.6


def test_append_of_no_rows_writes_nothing():
    """Sequences of padding alone, whatever their block's scale holds."""
    c = kv8.empty(2, 1, 64, 64)
    c.tensors[2].fill_(math.nan)
    before = snapshot(c)
    k = torch.randn(2, 3, 1, 64, device="cuda")
    kv8.append(c, k, k, ints([5, 37]), n_new=ints([0, -2]))
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(c.tensors, before))


# ---------------------------------------------------------------- attention
def fill(s, h, c, d, g, spread=1.0, weights=True):
    """A full cache with scales that differ from block to block."""
    k, v = (torch.randint(-127, 128, (s, h, c, d), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    ks, vs = (0.02 * torch.exp(spread * torch.randn(s, h, c // 16, generator=g, device="cuda")) for _ in range(2))
    acc = torch.rand(s, h, c, generator=g, device="cuda") if weights else None
    return kv8.Cache(k, v, ks, vs, acc)


def attend64(c, q, lens, n_new, causal, scale):
    """(out, bound on the error before the last rounding, weights drawn, bound on theirs)"""
    k8, v8, ks, vs, _ = c.tensors
    s, n, hq, d = q.shape
    h = k8.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    drawn = torch.zeros(k8.shape[:3], dtype=torch.float64, device="cuda")
    derr = torch.zeros_like(drawn)
    for b in range(s):
        m = min(max(lens[b], 0), k8.shape[2])
        nb = n if n_new is None else min(max(n_new[b], 0), n)
        if not m or not nb:
            continue
        for g in range(h):
            blocks = torch.arange(m, device="cuda") // 16
            k = k8[b, g, :m].double() * ks[b, g, blocks].double()[:, None]
            v = v8[b, g, :m].double() * vs[b, g, blocks].double()[:, None]
            x = q[b, :nb, g * (hq // h):(g + 1) * (hq // h)].double()            # [rows, group, d]
            sc = torch.matmul(x, k.T) * scale
            mag = torch.matmul(x.abs(), k.abs().T) * abs(scale)
            lim = torch.arange(nb, device="cuda")[:, None] + (m - nb + 1) if causal else torch.full((nb, 1), m, device="cuda")
            seen = (torch.arange(m, device="cuda") < lim)[:, None]
            sc = torch.where(seen, sc, -torch.inf)
            top = sc.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(sc - torch.where(top.isfinite(), top, 0.0)), 0.0)
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            # a score: d products summed in fp32 and three factors, (d + 8) u of its terms' magnitude (and, of rows held
            # as 11-bit numbers under a common power of two, d 2^-25 of the row's largest: less); its exponent in base 2:
            # 2 u of the score and of the maximum; a probability moves by the errors of its score, of the largest score
            # and of the mean one
            delta = (d + 16) * U * torch.where(seen, mag, 0.0).amax(-1, keepdim=True)
            rel = 3 * delta + 16 * U + m * U * 2.0 ** -3
            o = torch.matmul(p, v)
            out[b, :nb, g * (hq // h):(g + 1) * (hq // h)] = o
            # each probability (times its block's scale) is an 11-bit number; the sum of m terms in fp32
            # (many partial sums: m / 8 u), and numbers under 2^-14 of the row's largest keep an absolute 2^-25 of it
            err[b, :nb, g * (hq // h):(g + 1) * (hq // h)] = torch.matmul(p, v.abs()) * (rel + 2.0 ** -11) + \
                m * 2.0 ** -38 * v.abs().amax()
            drawn[b, g, :m] = p.sum((0, 1))
            derr[b, g, :m] = (p * rel).sum((0, 1)) + p.sum((0, 1)) * nb * (hq // h) * U
    return out, err, drawn, derr


def check_attend(c, q, lens, *, n_new=None, causal=True, scale=None, weights=None, dtype=None, max_len=0, out=None):
    weights = c.tensors[4] is not None if weights is None else weights
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    before = c.tensors[4].clone() if weights else None
    want, err, drawn, derr = attend64(c, q, [min(n, max_len) for n in lens] if max_len else lens, n_new, causal, scale)
    got = kv8.attend(c, q, ints(lens), n_new=None if n_new is None else ints(n_new), causal=causal, scale=scale,
                     weights=weights, dtype=dtype, max_len=max_len, out=out)
    t = got.dtype
    rows = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    if n_new is not None:
        rows = torch.arange(q.shape[1], device="cuda") < ints(n_new)[:, None]
    within(got[rows], want[rows], (err + (want.abs() + err) * HALF[t] + TINY[t])[rows])
    if weights:
        total = before.double() + drawn
        within(c.tensors[4], total, derr + total * U)
        assert torch.equal(c.tensors[4][drawn == 0], before[drawn == 0])
    return got


def query(s, n, hq, d, g, dtype, size=1.0):
    return (size * torch.randn(s, n, hq, d, generator=g, device="cuda")).to(dtype)


LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("h,group,d", [(2, 1, 128), (2, 2, 128), (1, 3, 64), (2, 4, 64), (1, 8, 128), (1, 16, 64), (1, 32, 128)])
def test_attend_one_row(h, group, d, dtype):
    """One new token of each of 15 sequences of every length around tile and block ends, in one call."""
    g = gen(h * 100 + group + d)
    c = fill(len(LENS), h, 304, d, g)
    check_attend(c, query(len(LENS), 1, h * group, d, g, dtype), LENS)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n,group,d", [(1, 2, 128), (1, 8, 64), (3, 5, 64), (2, 16, 128)])
def test_attend_few_rows_in_one_workgroup_or_several(n, group, d, weights):
    """Sequences up to 512 slots by one workgroup a head, or as far as the call is sized for more by several."""
    g = gen(n * 10 + group)
    lens = [0, 1, n, 63, 64, 65, 300, 511, 512, 700]
    c = fill(len(lens), 2, 1040, d, g, weights=weights)
    for dtype in T16:
        q = query(len(lens), n, 2 * group, d, g, dtype)
        check_attend(c, q, lens, max_len=512)
        check_attend(c, q, lens, max_len=513)
        check_attend(c, q, lens, n_new=[n, n, 0, n - 1, n, 1, n, n, n, n])


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n,h,group,d", [(2, 2, 2, 128), (5, 1, 3, 64), (7, 2, 4, 128), (16, 1, 2, 64), (17, 2, 1, 128), (33, 1, 2, 128),
                                         (64, 2, 2, 64), (70, 1, 5, 128), (129, 1, 2, 128), (200, 2, 1, 64), (3, 1, 32, 64)])
def test_attend_rows(n, h, group, d, weights):
    """Several new rows behind histories of all kinds of lengths, and a whole prompt."""
    g = gen(n * 100 + group)
    lens = [n, n + 1, n + 47, n + 64, n + 191, 512]
    c = fill(len(lens), h, 512, d, g, weights=weights)
    for dtype in T16:
        check_attend(c, query(len(lens), n, h * group, d, g, dtype), lens)


@pytest.mark.parametrize("n", [1, 3, 40, 150])
def test_attend_empty_rows_and_ragged_batches(n):
    """Sequences of no slots, rows that see none (fewer slots than rows), padded rows: 0, 0, left as they were."""
    g = gen(n)
    lens = [0, 1, n // 2, n, 255, -4, 1000]
    new = [n, n, n, 1, n - 1, n, 2 * n]
    c = fill(7, 2, 256, 128, g)
    q = query(7, n, 4, 128, g, torch.float16)
    out = torch.full_like(q, 7.0)
    got = check_attend(c, q, lens, n_new=new, out=out)
    assert got is out
    for b in range(7):
        nb = min(max(new[b], 0), n)
        m = min(max(lens[b], 0), 256)
        assert (out[b, nb:] == 7.0).all()
        assert (out[b, :max(nb - m, 0)] == 0).all()
    check_attend(c, q, lens, n_new=new, causal=False)
    check_attend(c, q, lens, n_new=[0] * 7)


@pytest.mark.parametrize("n", [1, 9, 100])
def test_attend_does_not_read_past_the_length(n):
    """Whatever stands behind a sequence's last slot (here the worst codes, and scales that are not finite)."""
    g = gen(n + 50)
    lens = [n, n + 5, 177]
    c = fill(3, 2, 320, 64, g)
    q = query(3, n, 4, 64, g, torch.bfloat16)
    first = check_attend(c, q, lens, weights=False)
    for b, m in enumerate(lens):
        c.tensors[0][b, :, m:] = -128
        c.tensors[1][b, :, m:] = -128
        for t, bad in zip(c.tensors[2:4], (math.nan, math.inf)):
            t[b, :, (m + 15) // 16:] = bad
    assert torch.equal(first, kv8.attend(c, q, ints(lens)))


@pytest.mark.parametrize("n", [1, 6, 90])
def test_attend_strides_types_and_scale(n):
    """Heads before rows, rows that are not 16-byte aligned, fp32 output, another scale, a bound on the lengths."""
    g = gen(n + 7)
    k = fill(2, 6, 256, 128, g)
    # every other head of a larger cache: strides of its own
    c = kv8.Cache(*(t[:, ::2] for t in k.tensors))
    wide = torch.randn(2, 6, n, 130, generator=g, device="cuda").half()
    q = wide[..., 1:129].transpose(1, 2)
    out = torch.zeros(2, 6, n, 131, device="cuda")[..., 1:129].transpose(1, 2)
    check_attend(c, q, [n, 256], out=out)
    check_attend(c, q, [n, 256], out=torch.zeros(2, 6, n, 136, device="cuda").bfloat16()[..., 8:].transpose(1, 2), scale=0.3)
    check_attend(c, q, [n, 256], dtype=torch.float32, scale=-0.05)
    check_attend(c, q, [n, 200], max_len=100 + n, dtype=torch.float32)


@pytest.mark.parametrize("n", [1, 4, 80])
def test_attend_large_and_sharp(n):
    """Scores of hundreds (a softmax that is one slot), of zero, values and scales far apart, rows that are not finite."""
    g = gen(n + 9)
    c = fill(2, 1, 192, 128, g, spread=3.0)
    for dtype in T16:
        q = query(2, n, 2, 128, g, dtype, size=20.0)
        check_attend(c, q, [192, n + 3])
        check_attend(c, q, [192, n + 3], scale=0.0)
        check_attend(c, torch.zeros_like(q), [192, n + 3])
        check_attend(c, (q.float() * 2.0 ** -30).to(dtype) if dtype == torch.bfloat16 else q * 0.001, [192, n + 3], scale=2.0 ** 20)
        q[0, 0, 1, 5] = math.nan
        q[1, n - 1, 0, 7] = math.inf
        got = kv8.attend(c, q, ints([192, n + 3]))
        bad = torch.zeros(2, n, 2, dtype=torch.bool, device="cuda")
        bad[0, 0, 1] = bad[1, n - 1, 0] = True
        assert got[bad].isnan().all() and not got[~bad].isnan().any()
    if n == 1:
        q = query(2, n, 2, 128, g, torch.bfloat16, size=3e37)       # past what 16 bits of fp16 hold
        check_attend(c, q, [192, 50], scale=1e-38)


@pytest.mark.parametrize("n", [1, 40])
def test_attend_smallest_queries(n):
    """Rows of fp16's subnormal numbers, and of bfloat16's, under a scale that makes scores of them."""
    g = gen(n + 90)
    c = fill(2, 1, 192, 128, g)
    tiny = (2.0 ** -22 * torch.randn(2, n, 2, 128, generator=g, device="cuda")).half()
    check_attend(c, tiny, [192, n + 3], scale=2.0 ** 21)
    check_attend(c, query(2, n, 2, 128, g, torch.bfloat16, 2.0 ** -128), [192, n + 3], scale=2.0 ** 126)


def test_attend_most_rows():
    """65,535 rows of 31 heads: rows find their token and head; all but the last see nothing or little."""
    g = gen(13)
    c = fill(1, 1, 32, 64, g)
    q = torch.randn(1, 65535, 31, 64, generator=g, device="cuda").half()
    check_attend(c, q, [29])
    check_attend(c, q, [17], causal=False, weights=False)


def test_attend_long():
    """One row over 40,001 slots of 8 heads, and 40 rows over them."""
    g = gen(11)
    c = fill(1, 8, 40016, 64, g, spread=0.3)
    for n in (1, 40):
        check_attend(c, query(1, n, 16, 64, g, torch.float16, 2.0), [40001])


@pytest.mark.parametrize("s,h,slots", [(1, 1, 700), (3, 8, 4001), (5, 8, 2500), (2, 5, 13000)])
def test_attend_many_rows_of_many_sizes(s, h, slots):
    """60 rows of two heads over few and many slot tiles: how many waves share a tile of the weights' pass, and into how many
    splits the slots go, changes with the size."""
    g = gen(slots)
    c = fill(s, h, -(-slots // 16) * 16, 128, g, spread=0.3)
    check_attend(c, query(s, 60, 2 * h, 128, g, torch.float16, 1.5), [slots - 37 * b for b in range(s)])


def test_attend_offsets_past_32_bits():
    """A head whose codes lie past 2^31 bytes, at slots past 2^31 bytes of it."""
    c = kv8.empty(1, 2, 17_000_000, 128)
    slots = c.shape[2]
    g = gen(12)
    k, v = (torch.randn(1, 33, 2, 128, generator=g, device="cuda") for _ in range(2))
    at = slots - 33
    kv8.append(c, k, v, ints([at]))
    q = query(1, 1, 4, 128, g, torch.float16, 3.0)
    # all other slots are zero codes of scale 0: score 0, value 0
    got = kv8.attend(c, q, ints([slots]), weights=True).double()
    k8, v8 = (x.double().transpose(1, 2) for x in kv8.read(c, ints([at]), 33, dtype=torch.float32))
    x = torch.matmul(q.double().transpose(1, 2).reshape(1, 2, 2, 128), k8.transpose(2, 3)) * 128 ** -0.5
    p = x.exp() / (x.exp().sum(-1, keepdim=True) + at)
    want = torch.matmul(p, v8).reshape(1, 1, 4, 128)
    # 4 u of each of many partial sums of the 17 million equal terms, 2^-11 of the probabilities
    within(got, want, torch.matmul(p, v8.abs()).reshape(1, 1, 4, 128) * 2.0 ** -9 + 2.0 ** -25)
    within(c.tensors[4][:, :, at:], p.sum(2), p.sum(2) * 2.0 ** -10)
    head = kv8.read(c, ints([at]), 33)[0]
    within(head, k.double(), (c.tensors[2][0, :, -3:].max() * 0.51).double())


@pytest.mark.parametrize("n", [1, 6, 12, 40, 150])
def test_attend_whatever_the_workspace_holds(n, monkeypatch):
    """Many splits, the last of them near the rows' own slots, and one: no part of it is read that was not written."""
    g = gen(n + 60)
    c = fill(1, 1, 5008, 128, g, spread=0.3)
    q = query(1, n, 1, 128, g, torch.float16, 2.0)

    def of_nan(*size, dtype=None, device=None):
        return torch.full(size, 0xff, dtype=dtype, device=device)

    want = [check_attend(c, q, [m]) for m in (4608 + 20, 4608 + n, 300)]
    monkeypatch.setattr(kv8.torch, "empty", of_nan)     # the workspace's
    got = [check_attend(c, q, [m]) for m in (4608 + 20, 4608 + n, 300)]
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("size", [1e-33, 1e-36, 1e-38])
def test_attend_tiny_values(n, size):
    """Value scales down to fp32's subnormal numbers."""
    g = gen(n + 70)
    c = fill(2, 1, 400, 128, g)
    c.tensors[3].mul_(size)
    q = query(2, n, 2, 128, g, torch.float16, 2.0)
    want, err, _, _ = attend64(c, q, [400, n + 7], None, True, 128 ** -0.5)
    got = kv8.attend(c, q, ints([400, n + 7]), dtype=torch.float32)
    # a probability times its scale is a multiple of 2^-24 at least of 2^-124: 127 * 2^-149 a slot; then the results'
    # own rounding, to multiples of 2^-149 too, in up to four sums
    within(got, want, err + want.abs() * U + (400 * 127 + 4) * 2.0 ** -149)


@pytest.mark.parametrize("n", [5, 12, 60])
def test_weights_of_rows_that_are_not_finite(n):
    """Such a row makes the weights of the slots that it sees NaN, and no others."""
    g = gen(n + 80)
    c = fill(2, 2, 256, 64, g)
    q = query(2, n, 4, 64, g, torch.float16)
    q[:, 1] = 0.0
    lens = [200, n]
    before = c.tensors[4].clone()
    kv8.attend(c, q, ints(lens), weights=True)
    clean = c.tensors[4].clone()
    q[0, 1, 0, 3] = math.nan            # of kv head 0
    q[1, 1, 3, 60] = math.inf           # of kv head 1
    c.tensors[4].copy_(before)
    kv8.attend(c, q, ints(lens), weights=True)
    seen = torch.zeros_like(clean, dtype=torch.bool)
    seen[0, 0, :lens[0] - n + 2] = True
    seen[1, 1, :2] = True
    assert c.tensors[4][seen].isnan().all()
    assert torch.equal(c.tensors[4][~seen], clean[~seen])


def test_attend_refusals():
    c = fill(2, 2, 64, 64, gen(1), weights=False)
    q = torch.randn(2, 3, 4, 64, device="cuda").half()
    lens = ints([10, 20])
    for bad in [dict(q=q.float()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(lens=ints([1])), dict(lens=lens.long()),
                dict(lens=lens.cpu()), dict(lens=None), dict(weights=True), dict(max_len=65), dict(out=q[:, :2]), dict(out=q.double()),
                dict(n_new=ints([1])), dict(scale=math.nan), dict(q=q.transpose(2, 3).contiguous().transpose(2, 3))]:
        a = dict(q=q, lens=lens) | bad
        with pytest.raises(kv8.Kv8Error):
            kv8.attend(c, a.pop("q"), a.pop("lens"), **a)
    with pytest.raises(kv8.Kv8Error):
        kv8.append(c, q[:, :, :2].float(), q[:, :, :2], lens)
    with pytest.raises(kv8.Kv8Error):
        kv8.append(c, q, q, lens)
    k = c.tensors
    for bad in [(k[0].short(), *k[1:]), (k[0], k[1][:, :1], *k[2:]), (k[0], k[1], k[2][..., :3], k[3], None),
                (k[0].transpose(2, 3), k[1].transpose(2, 3), *k[2:]), (k[0], k[1], k[2], k[3], k[2])]:
        with pytest.raises(kv8.Kv8Error):
            kv8.Cache(*bad)


# ---------------------------------------------------------------- eviction
def evict64(c, lens, keep, sink, recent):
    """Kept slots by the definition, as lists [sequence][head]."""
    acc = c.tensors[4].double().cpu().numpy()
    out = []
    for b in range(acc.shape[0]):
        m = min(max(lens[b], 0), acc.shape[2])
        row = []
        for h in range(acc.shape[1]):
            if m <= keep:
                row.append(list(range(m)))
                continue
            sure = [t for t in range(m) if t < sink or t >= m - recent]
            w = np.where(np.isnan(acc[b, h]), -np.inf, acc[b, h])
            rest = sorted(range(sink, m - recent), key=lambda t: (-w[t], t))[:keep - len(sure)]
            row.append(sorted(sure + rest))
        out.append(row)
    return out


def check_evict(c, lens, keep, sink, recent, room=None):
    s, h, slots, d = c.shape
    to = fill(s, h, room or -(-keep // 16) * 16, d, gen(99))
    before = snapshot(to)
    kept, left = kv8.evict(c, to, ints(lens), n_keep=keep, n_sink=sink, n_recent=recent)
    want = evict64(c, lens, keep, sink, recent)
    k8, v8, ks, vs, acc = (t.cpu() for t in c.tensors)
    for b in range(s):
        assert left[b].item() == len(want[b][0])
        for g in range(h):
            at = torch.tensor(want[b][g], dtype=torch.long)
            n = len(at)
            assert kept[b, g].tolist() == at.tolist() + [-1] * (keep - n)
            assert torch.equal(to.tensors[4][b, g, :n].cpu().nan_to_num(nan=-1.0), acc[b, g, at].nan_to_num(nan=-1.0))
            assert torch.equal(to.tensors[4][b, g, n:], before[4][b, g, n:])
            for codes, scales, got, gots, was in ((k8, ks, to.tensors[0], to.tensors[2], before[0]), (v8, vs, to.tensors[1], to.tensors[3], before[1])):
                assert torch.equal(got[b, g, n:], was[b, g, n:])
                s0 = scales[b, g, at // 16]
                for blk in range((n + 15) // 16):
                    mine = s0[blk * 16:blk * 16 + 16]
                    assert gots[b, g, blk].item() == mine.max().item()
                    # the ratio's rounding and the product's, of up to 127; then to the nearest whole number
                    exact = codes[b, g, at[blk * 16:blk * 16 + 16]].double() * (mine.double() / mine.max().clamp_min(1e-38).double())[:, None]
                    within(got[b, g, blk * 16:min(blk * 16 + 16, n)].cpu().float(), exact, 0.5 + 127 * 3 * U)
    return to, kept, left


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (16, 0, 16), (20, 4, 7), (33, 33, 0), (50, 0, 1), (100, 3, 90), (128, 10, 10)])
def test_evict(keep, sink, recent, d):
    c = fill(5, 2, 208, d, gen(keep))
    check_evict(c, [208, 129, 0, 33, 500], keep, sink, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "special"])
def test_evict_ties(kind):
    """Equal weights go to the lowest slots; -0 equals +0; NaN is the least, with -infinity."""
    g = gen(4)
    c = fill(2, 3, 3008, 64, g)
    acc = c.tensors[4]
    if kind == "equal":
        acc.fill_(0.25)
    elif kind == "few":
        acc.copy_(torch.randint(0, 3, acc.shape, generator=g, device="cuda").float())
    elif kind == "signs":
        acc.copy_(torch.randint(-1, 2, acc.shape, generator=g, device="cuda").float() * 0.0)
        acc[:, :, ::7] = -1e-40
        acc[:, :, ::11] = 1e-40
    else:
        acc.normal_(generator=g)
        acc[:, :, ::3] = math.nan
        acc[:, :, 1::5] = -math.inf
        acc[:, :, 2::9] = math.inf
    for keep in (100, 1500, 2900):
        check_evict(c, [3001, 2905], keep, 5, 60)


@pytest.mark.parametrize("n", [1023, 1025, 4096, 4097, 8192, 8200, 16384, 16390, 32768, 32771])
@pytest.mark.parametrize("kind", ["any", "close", "coarse"])
def test_evict_threshold(n, kind):
    """Lengths around the numbers of slots that a thread takes; weights that part at their first bytes, only at their
    last, or not at all."""
    g = gen(n)
    c = fill(1, 1, -(-n // 16) * 16, 64, g)
    if kind == "close":
        c.tensors[4].mul_(2.0 ** -10).add_(1.0)
    elif kind == "coarse":
        c.tensors[4].mul_(16.0).round_()
    check_evict(c, [n], n // 3, 3, n // 7)
    check_evict(c, [n], n // 3, n // 3 - 20, 20)


def test_evict_long_and_views():
    g = gen(6)
    big = fill(1, 4, 70000, 64, g)
    c = kv8.Cache(*(t[:, 1:3] for t in big.tensors))
    c.tensors[4].mul_(c.tensors[4]).mul_(c.tensors[4])
    check_evict(c, [69991], 41003, 4, 1000, room=41024)


def test_evict_refuses_its_own_memory():
    c = fill(1, 1, 64, 64, gen(1))
    with pytest.raises(kv8.Kv8Error, match="other memory"):
        kv8.evict(c, c, ints([64]), n_keep=10)
    with pytest.raises(kv8.Kv8Error, match="n_keep"):
        kv8.evict(c, fill(1, 1, 32, 64, gen(1)), ints([64]), n_keep=33)


def test_evict_writes_the_lengths_in_place():
    """len_out may be lens: every head reads the old length."""
    g = gen(8)
    c = fill(40, 8, 96, 64, g)
    lens = [96 - s for s in range(40)]
    to, kept, left = check_evict(c, lens, 33, 3, 5)
    at, again, mine = ints(lens), torch.empty_like(kept), fill(40, 8, 48, 64, gen(99))
    kv8._check(kv8.load_kv8_library().q3t_kv8_evict(c.index, c.ref, mine.ref, at.data_ptr(), 0, 33, 3, 5, again.data_ptr(),
                                                    at.data_ptr(), kv8._stream(c.index)), "evict")
    assert torch.equal(at, left) and torch.equal(again, kept)
    assert all(torch.equal(a, b) for a, b in zip(to.tensors, mine.tensors))


# ---------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_read(d, dtype):
    c = fill(3, 2, 96, d, gen(d))
    start, n = [0, 90, -5], 37
    got = kv8.read(c, ints(start), n, dtype=dtype)
    for x, codes, scales in zip(got, c.tensors[:2], c.tensors[2:4]):
        want = torch.zeros(3, n, 2, d, dtype=torch.float64, device="cuda")
        for b in range(3):
            for i in range(n):
                t = start[b] + i
                if 0 <= t < 96:
                    want[b, i] = codes[b, :, t].double() * scales[b, :, t // 16].double()[:, None]
        # the product in fp32, then the type
        within(x, want, want.abs() * (U + HALF[dtype] * (1 + U)) + TINY[dtype])
    assert kv8.read(c, ints(start), 0)[0].shape == (3, 0, 2, d)


# ---------------------------------------------------------------- together
def session(c, spare, x, lens, freq, gains, group):
    """A session's round: rotate new rows, store them, attend with weights kept, evict.  Returns what it computed."""
    s, n = x["q"].shape[:2]
    pos = (lens[:, None] + torch.arange(n, device="cuda", dtype=torch.int32) + 500).flatten().int()
    q, k = kv8.rope([x["q"].flatten(0, 1), x["k"].flatten(0, 1)], pos, freq, gains=gains, dtype=torch.float16)
    q, k = q.unflatten(0, (s, n)), k.unflatten(0, (s, n))
    kv8.append(c, k, x["v"], lens)
    o = kv8.attend(c, q, lens + n, weights=True)
    kept, left = kv8.evict(c, spare, lens + n, n_keep=96, n_sink=4, n_recent=32)
    return o, kept, left


def session_state(seed):
    g = gen(seed)
    x = {"q": torch.randn(3, 20, 8, 128, generator=g, device="cuda"), "k": torch.randn(3, 20, 4, 128, generator=g, device="cuda"),
         "v": torch.randn(3, 20, 4, 128, generator=g, device="cuda").half()}
    return fill(3, 4, 160, 128, g), fill(3, 4, 96, 128, gen(1)), x, ints([100, 3, 140])


def test_session_together():
    """The operators one after another, each checked on what the one before it wrote."""
    freq = torch.from_numpy(kv8.rope_freqs(128, 1e6, "turns", 2.0, 32768)).cuda()
    gains = [torch.full((128,), 1.1, device="cuda"), None]
    c, spare, x, lens = session_state(3)
    acc0 = c.tensors[4].clone()
    pos = (lens[:, None] + torch.arange(20, device="cuda") + 500).flatten().int()
    q, k = kv8.rope([x["q"].flatten(0, 1), x["k"].flatten(0, 1)], pos, freq, gains=gains, dtype=torch.float16)
    for y, xx, gain in ((q, x["q"], gains[0]), (k, x["k"], None)):
        w, m = rope64(xx.flatten(0, 1), pos, freq, gain, False, 1.0, 1e-6)
        within(y, w, rope_bound(w, m, torch.float16))
    k = k.unflatten(0, (3, 20))
    want = append64(c, k, x["v"], lens.tolist(), None)
    kv8.append(c, k, x["v"], lens)
    check_append(c, None, want, acc0)
    check_attend(c, q.unflatten(0, (3, 20)), [120, 23, 160])
    to, kept, left = check_evict(c, [120, 23, 160], 96, 4, 32)
    assert left.tolist() == [96, 23, 96]
    # attention goes on over what was kept
    check_attend(to, q.unflatten(0, (3, 20))[:, -1:], left.tolist())
    # and all of it at once gives the same bits
    c2, spare2, x2, lens2 = session_state(3)
    o, kept2, left2 = session(c2, spare2, x2, lens2, freq, gains, 2)
    assert torch.equal(kept2, kept) and torch.equal(left2, left)
    for a, b in zip(c2.tensors, c.tensors):
        assert torch.equal(a, b)


def test_two_graphs_and_streams():
    """Two captured sessions replayed on two streams at once, with eager sessions between the replays: every replay
    equals the eager result (a call's workspace is its own)."""
    freq = torch.from_numpy(kv8.rope_freqs(128, 1e6)).cuda()
    gains = [None, None]
    states = [session_state(s) for s in (5, 6)]
    wants = []
    for s in (5, 6):
        st = session_state(s)
        out = session(*st, freq, gains, 2)
        wants.append(([t.clone() for t in out], snapshot(st[0]), snapshot(st[1])))
    firsts = [(snapshot(st[0]), snapshot(st[1])) for st in states]
    streams = [torch.cuda.Stream() for _ in states]
    graphs, outs = [], []
    for st, stream in zip(states, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(session(*st, freq, gains, 2))
        graphs.append(g)
    for _ in range(3):
        for st, first in zip(states, firsts):
            for c, f in zip(st[:2], first):
                for t, u in zip(c.tensors, f):
                    t.copy_(u)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        eager = session_state(7)
        session(*eager, freq, gains, 2)
        torch.cuda.synchronize()
        for st, out, (want, cw, sw) in zip(states, outs, wants):
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            for a, b in zip(st[0].tensors + st[1].tensors, cw + sw):
                assert torch.equal(a, b)


def test_current_device_and_side_stream():
    """Calls leave the current device as it was and run on torch's current stream."""
    c = fill(1, 2, 64, 64, gen(1))
    q = query(1, 1, 2, 64, gen(2), torch.float16)
    want = kv8.attend(c, q, ints([50]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv8.attend(c, q, ints([50]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.cuda.current_device() == 0 and torch.equal(got, want)
