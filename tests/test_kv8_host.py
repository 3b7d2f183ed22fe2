"""The 8-bit cache operators' C ABI on the host: what the header declares is
bound and exported, structs match, refusals come before any device work (no
GPU here), and the rotary frequencies."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

from qwen3_tts_amd import kv8
from qwen3_tts_amd.device import LIB_PATH

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "q3t_kv8.h")


def header():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_declares_the_bound_functions():
    declared = sorted(set(re.findall(r"\b(q3t_kv8_[a-z_0-9]+)\s*\(", header())))
    assert declared == sorted(kv8.KV8_EXPORTS)
    lib = ctypes.CDLL(LIB_PATH)
    assert not [f for f in declared if not hasattr(lib, f)]


@pytest.mark.parametrize("name,cls", [("q3t_kv8", kv8.CCache), ("q3t_kv8_rope_rows", kv8.CRopeRows),
                                      ("q3t_kv8_attend_args", kv8.CAttendArgs)])
def test_structs_match_the_header(name, cls):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header(), re.S).group(1)
    names = []
    for line in body.split(";"):
        names += [re.search(r"([a-z_0-9]+)\s*$", part).group(1) for part in line.split(",") if part.strip()]
    assert names == [n for n, _ in cls._fields_]


# addresses that are never followed: every call below is refused first, or has nothing to do
P = 4096


def cache(**kw):
    c = kv8.CCache(P, P, P, P, P, 1 << 20, 1 << 16, 64, 32, 1024, 512, 2, 2, 512, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attend_args(**kw):
    a = kv8.CAttendArgs(P, P, 512, 256, 128, 512, 256, 128, 1, 1, 1, 4, P, 0, None, 0, 1, 0.1, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHES = [({"k": None}, "null"), ({"vs": None}, "null"), ({"head_dim": 96}, "head_dim"), ({"n_slots": 40}, "n_slots"),
              ({"n_slots": 0}, "n_slots"), ({"n_seq": 0}, "n_seq"), ({"n_kv_head": 0}, "n_kv_head"), ({"k": P + 8}, "aligned"),
              ({"head": 24}, "aligned")]


def refused(rc, what):
    assert rc < 0
    message = kv8.load_kv8_library().q3t_kv8_last_error().decode()
    assert what in message, message


@pytest.mark.parametrize("change,what", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(change, what):
    lib, c, good = kv8.load_kv8_library(), cache(**change), cache()
    b = ctypes.byref
    refused(lib.q3t_kv8_append(0, b(c), P, P, 0, 0, 0, 0, 1, None, 0, None, None), what)
    refused(lib.q3t_kv8_attend_ws(b(c), b(attend_args())), what)
    refused(lib.q3t_kv8_attend(0, b(c), b(attend_args()), P, 1 << 40, None), what)
    refused(lib.q3t_kv8_evict(0, b(c), b(good), None, 0, 1, 0, 0, P, None, None), what)
    refused(lib.q3t_kv8_evict(0, b(good), b(c), None, 0, 1, 0, 0, P, None, None), what)
    refused(lib.q3t_kv8_read(0, b(c), None, 0, 1, 0, P, P, None), what)


@pytest.mark.parametrize("change,what", [({"q_type": 0}, "q must be"), ({"o_type": 8}, "out must be"), ({"n_rows": -1}, "n_rows"),
                                         ({"n_head": 3}, "n_head"), ({"n_head": 128}, "n_head"), ({"max_len": 513}, "max_len"),
                                         ({"max_len": -1}, "max_len"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"),
                                         ({"q": None}, "null rows")])
def test_attend_refuses(change, what):
    lib = kv8.load_kv8_library()
    refused(lib.q3t_kv8_attend(0, ctypes.byref(cache()), ctypes.byref(attend_args(**change)), P, 1 << 40, None), what)


def test_attend_refuses_weights_without_acc_and_a_small_workspace():
    lib, b = kv8.load_kv8_library(), ctypes.byref
    refused(lib.q3t_kv8_attend_ws(b(cache(acc=None)), b(attend_args())), "weights")
    assert lib.q3t_kv8_attend_ws(b(cache(acc=None)), b(attend_args(weights=0))) >= 0
    # one workgroup a head takes up to 512 slots, with no workspace
    assert lib.q3t_kv8_attend_ws(b(cache()), b(attend_args())) == 0
    more = cache(n_slots=1024)
    need = lib.q3t_kv8_attend_ws(b(more), b(attend_args()))
    assert need > 0
    refused(lib.q3t_kv8_attend(0, b(more), b(attend_args()), P, need - 1, None), "workspace")
    refused(lib.q3t_kv8_attend(0, b(more), b(attend_args()), None, need, None), "workspace")
    refused(lib.q3t_kv8_attend(0, b(more), b(attend_args()), P + 4, need, None), "aligned")


def test_append_evict_read_refuse():
    lib, b = kv8.load_kv8_library(), ctypes.byref
    refused(lib.q3t_kv8_append(0, b(cache()), P, P, 8, 0, 0, 0, 1, None, 0, None, None), "type")
    refused(lib.q3t_kv8_append(0, b(cache()), None, P, 0, 0, 0, 0, 1, None, 0, None, None), "null")
    refused(lib.q3t_kv8_append(0, b(cache()), P, P, 0, 0, 0, 0, -1, None, 0, None, None), "n_rows")
    to = cache(k=P * 2, v=P * 2, ks=P * 2, vs=P * 2, acc=P * 2)

    def evict(f, t, keep, sink, recent, kept=P):
        return lib.q3t_kv8_evict(0, b(f), b(t), None, 0, keep, sink, recent, kept, None, None)
    refused(evict(cache(), cache(), 10, 1, 1), "other memory")
    refused(evict(cache(), to, 0, 0, 0), "n_keep")
    refused(evict(cache(), to, 513, 0, 0), "n_keep")
    refused(evict(cache(), to, 10, 5, 6), "n_sink")
    refused(evict(cache(), to, 10, -1, 6), "n_sink")
    refused(evict(cache(), to, 10, 0, 0, None), "kept")
    refused(evict(cache(acc=None), to, 10, 0, 0), "weights")
    refused(evict(cache(n_kv_head=1), to, 10, 0, 0), "same")
    refused(lib.q3t_kv8_read(0, b(cache()), None, 0, -1, 0, P, P, None), "n_rows")
    refused(lib.q3t_kv8_read(0, b(cache()), None, 0, 1, 2, P, P, None), "type")
    refused(lib.q3t_kv8_read(0, b(cache()), None, 0, 1, 0, P + 8, P, None), "aligned")


def test_sizes_past_a_launch_are_refused():
    lib, b = kv8.load_kv8_library(), ctypes.byref
    refused(lib.q3t_kv8_attend_ws(b(cache(n_slots=(1 << 29) + 16)), b(attend_args())), "n_slots")
    refused(lib.q3t_kv8_attend_ws(b(cache(n_seq=65535, n_kv_head=129)), b(attend_args())), "n_seq * n_kv_head")
    assert lib.q3t_kv8_attend_ws(b(cache(n_slots=1 << 29)), b(attend_args(max_len=1 << 29))) > 0
    refused(lib.q3t_kv8_append(0, b(cache()), P, P, 0, 0, 0, 0, (1 << 26) + 1, None, 0, None, None), "n_rows")
    refused(lib.q3t_kv8_read(0, b(cache()), None, 0, 1 << 27, 0, P, P, None), "n_rows")
    rows = (kv8.CRopeRows * 1)(kv8.CRopeRows(P, 2 * P, 256, 128, 256, 128, None, 2, 0, 1))
    refused(rope_call(rows, tokens=(1 << 26) + 1), "n_tokens")


def rope_call(rows, n=1, tokens=4, d=128, rot=128, freq=P):
    return kv8.load_kv8_library().q3t_kv8_rope(0, rows, n, tokens, d, rot, 0, None, 0, freq, 1.0, 1e-6, None)


def test_rope_refuses():
    def rows(**kw):
        r = (kv8.CRopeRows * 4)(*[kv8.CRopeRows(P, 2 * P, 256, 128, 256, 128, None, 2, 0, 1) for _ in range(4)])
        for k, v in kw.items():
            setattr(r[0], k, v)
        return r
    refused(rope_call(rows(), n=0), "tensors")
    refused(rope_call(rows(), n=5), "tensors")
    refused(rope_call(rows(), d=24), "head_dim")
    refused(rope_call(rows(), d=272), "head_dim")
    refused(rope_call(rows(), rot=63), "rot_dim")
    refused(rope_call(rows(), rot=130), "rot_dim")
    refused(rope_call(rows(), rot=0), "rot_dim")
    refused(rope_call(rows(), tokens=-1), "n_tokens")
    refused(rope_call(rows(), freq=None), "null")
    refused(rope_call(rows(x=None)), "null")
    refused(rope_call(rows(x_type=8)), "types")
    refused(rope_call(rows(n_head=0)), "n_head")
    refused(rope_call(rows(y=P)), "in place")
    refused(rope_call(rows(y=P, y_type=0, y_token=512)), "in place")


def test_nothing_to_do_is_no_error():
    lib, b = kv8.load_kv8_library(), ctypes.byref
    assert rope_call((kv8.CRopeRows * 1)(kv8.CRopeRows(None, None, 0, 0, 0, 0, None, 2, 0, 0)), tokens=0) == 0
    assert lib.q3t_kv8_append(0, b(cache()), None, None, 0, 0, 0, 0, 0, None, 0, None, None) == 0
    assert lib.q3t_kv8_attend(0, b(cache()), b(attend_args(n_rows=0, q=None, out=None)), None, 0, None) == 0
    assert lib.q3t_kv8_read(0, b(cache()), None, 0, 0, 0, None, None, None) == 0


def test_no_device_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    lib, b = kv8.load_kv8_library(), ctypes.byref
    refused(lib.q3t_kv8_read(0, b(cache()), None, 0, 1, 0, P, P, None), "HIP device")


def test_cpu_tensors_are_refused():
    k = torch.zeros(1, 2, 32, 64, dtype=torch.int8)
    s = torch.zeros(1, 2, 2)
    with pytest.raises(kv8.Kv8Error):
        kv8.Cache(k, k, s, s)


@pytest.mark.parametrize("rot", [2, 8, 64, 128, 130])
@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_frequencies(rot, theta):
    i = np.arange(rot // 2)
    plain = theta ** (-2.0 * i / rot)
    np.testing.assert_allclose(kv8.rope_freqs(rot, theta), plain, rtol=1e-14)
    np.testing.assert_allclose(kv8.rope_freqs(rot, theta, "linear", 4.0), plain / 4, rtol=1e-14)
    if rot > 2:
        wide = (theta * 4.0 ** (rot / (rot - 2))) ** (-2.0 * i / rot)
        np.testing.assert_allclose(kv8.rope_freqs(rot, theta, "base", 4.0), wide, rtol=1e-13)
        # the slowest pair turns 4 times as slowly, the fastest as it did
        np.testing.assert_allclose(wide[-1], plain[-1] / 4, rtol=1e-12)
    f = kv8.rope_freqs(rot, theta, "turns", 4.0, 32768)
    turns = 32768 * plain / (2 * math.pi)
    # kept as they are: the unscaled call's own values (another library's power may differ in the last bit)
    assert np.all(f[turns >= 32.001] == kv8.rope_freqs(rot, theta)[turns >= 32.001])
    np.testing.assert_allclose(f[turns <= 1], plain[turns <= 1] / 4, rtol=1e-14)
    assert np.all((f <= plain * (1 + 1e-14)) & (f >= plain / 4 * (1 - 1e-14))) and np.all(np.diff(f) < 0)


def test_frequencies_refuse():
    for args, what in [((3, 1e4), "rot_dim"), ((258, 1e4), "rot_dim"), ((64, 0.0), "theta"), ((64, math.inf), "theta"),
                       ((64, 1e4, "linear", 0.5), "factor"), ((64, 1e4, "turns", 2.0, 0), "n_trained"), ((2, 1e4, "base", 2.0), "rot_dim")]:
        with pytest.raises(kv8.Kv8Error, match=what):
            kv8.rope_freqs(*args)
    with pytest.raises(kv8.Kv8Error):
        kv8.rope_freqs(64, 1e4, "other")
