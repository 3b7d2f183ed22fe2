"""The talker on an 8-bit cache (q3t_dev_kv_set_type I8): against the F16 cache
over the same history, its positions, its evictions, and the frame loop
past the end of the cache."""
import numpy as np
import pytest

from qwen3_tts_amd import config as qcfg
from qwen3_tts_amd import driver
from qwen3_tts_amd import kv8
from qwen3_tts_amd.device import Device, DeviceError
from qwen3_tts_amd.synth import Weights

pytestmark = pytest.mark.gpu
F16, BF16, I8 = 1, 30, 24


def device(wtype, kv, n_ctx=256, cfg=None, seed=7):
    cfg = cfg or qcfg.tiny()
    dev = Device(cfg)
    dev.upload_weights(Weights(cfg, wtype, seed=seed))
    dev.kv_set_type(kv)
    dev.kv_reserve(n_ctx)
    return dev


def rows(cfg, n, seed=0):
    return (np.random.default_rng(seed).standard_normal((n, cfg.hidden_size)) * 0.5).astype(np.float32)


def history(cfg, n, seed):
    rng = np.random.default_rng(seed)
    return [[rng.standard_normal((n, cfg.n_kv_head, cfg.head_dim)).astype(np.float16) for _ in range(2)] for _ in range(cfg.n_layers)]


def close(a, b, tol):
    """within tol of the row's largest magnitude"""
    worst = np.abs(a - b).max() / np.abs(b).max()
    assert worst <= tol, worst


# An attention output is an average of values, so it moves by at most what the values and probabilities move: values of
# the same history rounded to fp16 (2^-11), probabilities in 11 bits (2^-11 here, 2^-11 there), the rotated q rounded to fp16
# from fp32 angles of another table (2^-11 of a score of at most about 8: 2^-8), and the new rows' own
# quantisation, 1 / 254 of their block's largest value at n of n_past + n slots: together under 2^-6 of the values' size.  Two
# layers, each adding its output to a residual row of its own size or larger: 2^-5 bounds the hidden row, and for
# Q8_0 layers a quantisation step of the next input, 1 / 127 of a block's largest value, on top.
TOL = 2.0 ** -5 + 1 / 127


@pytest.mark.parametrize("wtype", ["q8_0", "f16"])
@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("n", [1, 2, 7, 70])
def test_matches_f16_cache_over_the_same_history(wtype, fast, n, monkeypatch):
    """The 8-bit cache's values (read back) as an F16 cache's history: the same step and prefill come out."""
    if fast:
        monkeypatch.delenv("Q3T_PF_EXACT", raising=False)
    cfg = qcfg.tiny()
    past = 151
    a, b = device(wtype, I8), device(wtype, F16)
    for layer, (k, v) in enumerate(history(cfg, past, 3)):
        a.kv_write(layer, k, v)
        k8, v8, w = a.kv_read(layer, 0, past)
        step = np.abs(k8 - k.astype(np.float32)).max()
        assert 0 < step <= np.abs(k).max() / 127 * 0.51 and not w.any()
        b.kv_write(layer, k8.astype(np.float16), v8.astype(np.float16))
    x = rows(cfg, n, 5)
    if n == 1:
        la, ha = a.talker_step(x[0], past)
        lb, hb = b.talker_step(x[0], past)
    else:
        ha, la = a.prefill(x, past)
        hb, lb = b.prefill(x, past)
    close(ha, hb, TOL)
    close(la, lb, TOL)
    # each head's probabilities sum to one for each row: the weights drawn add up to rows x heads
    for layer in range(cfg.n_layers):
        w = a.kv_read(layer, 0, past + n)[2]
        np.testing.assert_allclose(w.sum(1), n * cfg.n_head / cfg.n_kv_head, rtol=1e-5)
    a.close()
    b.close()


@pytest.mark.parametrize("wtype", ["q8_0", "f16"])
def test_prefill_in_parts_and_steps(wtype):
    """One prefill, the same rows in parts, and row by row: the same cache but for roundings."""
    cfg = qcfg.tiny()
    x = rows(cfg, 75, 2)
    whole, parts, steps = (device(wtype, I8) for _ in range(3))
    hw, lw = whole.prefill(x, 0)
    at = 0
    for n in (1, 2, 3, 66, 3):
        hp, lp = parts.prefill(x[at:at + n], at)
        at += n
    for i in range(75):
        ls, hs = steps.talker_step(x[i], i)
    # a block's earlier rows may be rounded again as its scale grows: two steps of 1 / 127 at most where rows are
    # stored one by one, on top of what the other paths differ by
    close(hp[-1], hw[-1], TOL + 2 / 127)
    close(hs, hw[-1], TOL + 2 / 127)
    kw, ks = whole.kv_read(0, 0, 75)[0], steps.kv_read(0, 0, 75)[0]
    assert np.abs(kw - ks).max() <= 3 * np.abs(kw).max() / 127
    for d in (whole, parts, steps):
        d.close()


def rotate(k, pos, freq):
    h = len(freq)
    c, s = np.cos(pos * freq), np.sin(pos * freq)
    return np.concatenate([k[..., :h] * c - k[..., h:] * s, k[..., h:] * c + k[..., :h] * s], -1)


@pytest.mark.parametrize("scaling", [None, (1, 8.0), (3, 16.0)])
def test_positions(scaling):
    """The key of layer 0 stored for a row at position p is the one at position 0 turned by p, also after evictions
    (p past the cache's slots) and with scaled frequencies."""
    cfg = qcfg.tiny()
    dev = device("f16", I8, 64)
    if scaling:
        dev.set_rope_scaling(*scaling)
        freq = kv8.rope_freqs(cfg.head_dim, cfg.rope_theta, {1: "linear", 3: "turns"}[scaling[0]], scaling[1], 32768)
    else:
        freq = kv8.rope_freqs(cfg.head_dim, cfg.rope_theta)
    x = rows(cfg, 1, 9)[0]
    dev.talker_step(x, 0)
    k0 = dev.kv_read(0, 0, 1)[0][0].astype(np.float64)
    pos = 1
    for _ in range(6):
        dev.prefill(rows(cfg, 48, pos), pos)
        pos += 48
        dev.kv_evict(pos, 10, 2, 4)
        assert np.abs(dev.kv_read(0, 0, 1)[0][0] - k0).max() <= np.abs(k0).max() / 60     # the sink stays
    dev.talker_step(x, pos)
    kp = dev.kv_read(0, 10, 1)[0][0]
    # both rows are off by half a step of their blocks' largest values (other rows share the later one)
    big = np.abs(dev.kv_read(0, 0, 11)[0]).max()
    assert np.abs(kp - rotate(k0, pos, freq)).max() <= 2 * big / 127
    dev.close()


@pytest.mark.parametrize("wtype", ["q8_0", "f16"])
def test_eviction_keeps_what_it_says(wtype):
    """Kept slots are the sinks, the last ones and those with the most weight; their values stay; the next step is that of a
    cache that was given these rows (rotation switched off, so that their positions do not matter)."""
    cfg = qcfg.tiny()
    a, b = device(wtype, I8), device(wtype, I8)
    for d in (a, b):
        d.set_rope_scaling(1, 1e30)
    x = rows(cfg, 141, 4)
    a.prefill(x[:140], 0)
    before = [a.kv_read(layer, 0, 140) for layer in range(cfg.n_layers)]
    kept = a.kv_evict(140, 60, 4, 16)
    for layer in range(cfg.n_layers):
        k, v, w = before[layer]
        kk, vv, ww = a.kv_read(layer, 0, 60)
        for h in range(cfg.n_kv_head):
            at = kept[layer, h]
            mid = sorted(range(4, 124), key=lambda t: (-w[h, t], t))[:40]
            assert at.tolist() == sorted([0, 1, 2, 3] + mid + list(range(124, 140)))
            assert np.array_equal(ww[h], w[h, at])
            # rounded to the new block's scale, at most the largest of the old ones
            assert np.abs(kk[:, h] - k[at, h]).max() <= 0.51 * np.abs(k[:, h]).max() / 127
            assert np.abs(vv[:, h] - v[at, h]).max() <= 0.51 * np.abs(v[:, h]).max() / 127
        b.kv_write(layer, kk.astype(np.float16), vv.astype(np.float16))
    la, ha = a.talker_step(x[140], 140)
    lb, hb = b.talker_step(x[140], 60)
    close(ha, hb, TOL)
    close(la, lb, TOL)
    assert np.array_equal(a.kv_read(0, 60, 1)[2] > 0, np.ones((cfg.n_kv_head, 1), bool))
    # fewer slots than asked for: nothing moves
    assert a.kv_evict(141, 61, 0, 0).tolist() == [[list(range(61))] * cfg.n_kv_head] * cfg.n_layers
    a.close()
    b.close()


@pytest.mark.parametrize("wtype", ["q8_0", "f16"])
def test_frame_loop_goes_past_the_cache(wtype):
    """40 greedy frames behind 20 rows in a cache of 48 slots, evicted between runs: the same codes and cache each time, the
    same codes in other chunks up to the first eviction (after 20 frames here, 28 there), and the driver's loop."""
    cfg = qcfg.tiny()
    x, trailing = rows(cfg, 20, 6), rows(cfg, 3, 7)
    pad = rows(cfg, 1, 8)[0]

    def loop(chunks, keep):
        dev = device(wtype, I8, 48)
        dev.prefill(x, 0, want_hidden=False)
        dev.frames_begin(trailing, pad, 20, 40, eos_bias=-1e4)
        out, pos, evicted = [], 20, 0
        for n in chunks:
            if pos - evicted + n > 48:
                dev.kv_evict(pos, keep, 2, 8)
                evicted = pos - keep
            codes, eos = dev.frames_run(n)
            assert len(codes) == n and not eos
            out.append(codes)
            pos += n
        _, _, path = dev.frames_stats()
        assert path == 0
        left = dev.kv_read(0, 0, pos - evicted)
        dev.close()
        return np.concatenate(out), left

    a, left = loop([10, 10, 10, 10], 24)
    b, again = loop([10, 10, 10, 10], 24)
    assert np.array_equal(a, b) and all(np.array_equal(p, q) for p, q in zip(left, again))
    c, _ = loop([5, 5, 1, 17, 12], 24)
    assert np.array_equal(a[:20], c[:20])
    assert a.min() >= 0 and a[:, 0].max() < cfg.codec_vocab and a[:, 1:].max() < cfg.cp_vocab
    # the driver's bounded generate() is this loop
    dev = device(wtype, I8, 48)
    g = driver.generate(dev, cfg, None, max_len=40, temperature=0.0, eos_bias=-1e4, chunk=10, prefill_rows=(x, trailing, pad),
                        bound=(24, 2, 8))
    assert np.array_equal(g, a)
    dev.close()


def test_frames_after_the_end_leave_the_cache_alone():
    """Frames past EOS run no step: neither the cache nor its weights move."""
    cfg = qcfg.tiny()
    dev = device("q8_0", I8, 64)
    dev.prefill(rows(cfg, 12, 1), 0, want_hidden=False)
    dev.frames_begin(rows(cfg, 1, 2), rows(cfg, 1, 3)[0], 12, 20, eos_bias=1e4, target_frames=0)
    codes, eos = dev.frames_run(4)
    n = 12 + len(codes)
    before = dev.kv_read(1, 0, 40)
    dev.frames_run(4)
    after = dev.kv_read(1, 0, 40)
    if eos:
        assert all(np.array_equal(p, q) for p, q in zip(before, after)), n
    dev.close()


def test_restart_and_switches():
    cfg = qcfg.tiny()
    dev = device("q8_0", I8, 64)
    x = rows(cfg, 50, 1)
    _, first = dev.prefill(x, 0)
    dev.kv_evict(50, 20, 2, 4)
    dev.talker_step(x[0], 50)
    # position 0 starts the cache anew, evictions forgotten
    _, again = dev.prefill(x, 0)
    assert np.array_equal(first, again)
    # the other types after it, and back
    dev.kv_set_type(F16)
    ref = device("q8_0", F16, 64)
    _, l0 = dev.prefill(x, 0)
    _, l1 = ref.prefill(x, 0)
    assert np.array_equal(l0, l1)
    dev.kv_set_type(I8)
    _, again = dev.prefill(x, 0)
    assert np.array_equal(first, again)
    # a long context: no bound but memory
    dev.kv_reserve(100_000)
    assert dev.lib.q3t_dev_kv_capacity(dev.h) == 100_000
    dev.prefill(x, 99_000)
    dev.talker_step(x[0], 99_999)
    dev.close()
    ref.close()


def test_streams_reserved_before_the_type_changed():
    """Streams hold F16 caches: not begun, written or prefilled while the type is I8, and as before after it."""
    cfg = qcfg.tiny()
    dev = device("q8_0", F16, 64)
    x = rows(cfg, 12, 3)
    dev.streams_reserve(2, 64)
    codes = []
    for kind in (F16, I8, F16):
        dev.kv_set_type(kind)
        args = [dict(trailing=x[:2], tts_pad=x[4], n_past=10, max_len=6), dict(trailing=x[:3], tts_pad=x[5], n_past=12, max_len=6)]
        if kind == I8:
            for call in (lambda: dev.stream_prefill(0, x), lambda: dev.streams_begin(args)):
                with pytest.raises(DeviceError, match="multi-stream"):
                    call()
            continue
        dev.stream_prefill(0, x[:10])
        dev.stream_prefill(1, x)
        dev.streams_begin(args)
        codes.append(dev.streams_run(6))
    for a, b in zip(*(c[0] for c in codes)):
        assert np.array_equal(a, b)
    dev.close()


def test_writing_no_rows_changes_nothing():
    cfg = qcfg.tiny()
    dev = device("q8_0", I8, 64)
    dev.prefill(rows(cfg, 50, 1), 0)
    dev.kv_evict(50, 20, 2, 4)
    none = np.zeros((0, cfg.n_kv_head, cfg.head_dim), np.float16)
    dev.kv_write(0, none, none)
    with pytest.raises(DeviceError, match="eviction"):
        dev.talker_step(rows(cfg, 1, 2)[0], 30)
    dev.talker_step(rows(cfg, 1, 2)[0], 50)
    dev.close()


def test_refusals():
    cfg = qcfg.tiny()
    dev = device("q8_0", I8, 64)
    x = rows(cfg, 60, 1)
    for call, what in [(lambda: dev.set_attn_capture(0), "capture"), (lambda: dev.streams_reserve(2, 64), "multi-stream"),
                       (lambda: dev.kv_set_type(8), "KV type"), (lambda: dev.prefill(x, 5), "Context length"),
                       (lambda: dev.talker_step(x[0], 64), "Context length"), (lambda: dev.talker_step(x[0], -1), "Context length"),
                       (lambda: dev.kv_evict(65, 10), "n_past"), (lambda: dev.kv_evict(30, 0), "n_keep"),
                       (lambda: dev.kv_evict(30, 65), "n_keep"), (lambda: dev.kv_evict(30, 10, 6, 5), "n_keep"),
                       (lambda: dev.kv_read(9, 0, 1), "out of range"), (lambda: dev.kv_read(0, 60, 5), "out of range"),
                       (lambda: dev.set_rope_scaling(7), "scaling"), (lambda: dev.set_rope_scaling(1, 0.5), "factor"),
                       (lambda: dev.set_rope_scaling(1, 2.0, 32768, 0.0), "mscale"), (lambda: dev.time_kernel(4, 1), "attention")]:
        with pytest.raises(DeviceError, match=what):
            call()
    dev.prefill(x, 0)
    dev.kv_evict(60, 20)
    with pytest.raises(DeviceError, match="eviction"):
        dev.talker_step(x[0], 59)
    dev.frames_begin(x[:1], x[1], 60, 100)
    with pytest.raises(DeviceError, match="Context length"):
        dev.frames_run(45)
    assert len(dev.frames_run(44)[0]) <= 44
    dev.close()
    f16 = device("q8_0", F16, 64)
    for call in (lambda: f16.kv_evict(10, 5), lambda: f16.kv_read(0, 0, 1), lambda: f16.set_rope_scaling(1, 2.0)):
        with pytest.raises(DeviceError, match="I8"):
            call()
    f16.set_attn_capture(0)
    with pytest.raises(DeviceError, match="capture"):
        f16.kv_set_type(I8)
    f16.close()
