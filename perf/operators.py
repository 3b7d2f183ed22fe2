"""The operators of a bounded 8-bit attention cache, as a program of this framework uses them.

Rotary positions (with the head norm that goes before them), rows quantised into the cache, attention over the
cache, eviction by accumulated attention weight, and the cached values read back.  A cache of S sequences, H key/value
heads, C slots and D dims is int8 codes k, v [S][H][C][D] and fp32 scales ks, vs [S][H][C / 16], one for each block
of 16 slots of a head (value = code * scale), with the attention weight each slot has drawn, acc [S][H][C].

Shapes follow the package's talker (16 query heads, 8 key/value heads of 128, 12.5 positions a second) and, with other
head layouts, what else such a cache is kept for.  Where `own` is false, run() computes in elementary torch operations;
where it is true it calls qwen3_tts_amd.kv8.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-tts.cpp_amd"))

own = False

BLOCK = 16             # slots that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one talker step: the query and key heads of one position, normed and rotated; a latency-bound call
        {"name": "rope_step", "op": "rope", "tokens": 1, "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128,
         "from": "f32", "to": "f16", "inter": False, "norm": True, "factor": 1.0, "far": 12000},
        # the long-context prompt of the package's configuration tests, one row past full tiles
        {"name": "rope_prompt_2049", "op": "rope", "tokens": 2049, "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128,
         "from": "f32", "to": "f16", "inter": False, "norm": True, "factor": 1.0, "far": 0},
        # neighbouring pairs, the first half of the head only, positions far beyond the trained ones, scaled
        {"name": "rope_far_11301", "op": "rope", "tokens": 11301, "heads": 32, "kv_heads": 4, "dim": 128, "rot": 64,
         "from": "bf16", "to": "bf16", "inter": True, "norm": False, "factor": 16.0, "far": 500000},
        # a frame of 16 streams: one new row each, at positions of their own inside begun blocks
        {"name": "append_step_16", "op": "append", "seqs": 16, "kv_heads": 8, "dim": 128, "rows": 1, "lo": 128,
         "hi": 2048, "from": "f32"},
        # the long-context prompt's rows behind a cached voice prompt that ends inside a block
        {"name": "append_prompt_2049", "op": "append", "seqs": 1, "kv_heads": 8, "dim": 128, "rows": 2049, "lo": 37,
         "hi": 37, "from": "f16"},
        # one stream's step in the middle of an utterance, weights kept for a later eviction
        {"name": "attend_step_2049", "op": "attend", "seqs": 1, "heads": 16, "kv_heads": 8, "dim": 128, "rows": 1,
         "lo": 2049, "hi": 2049, "type": "f16", "weights": True},
        # a server's frame: 16 streams, from a short prompt to a long reading
        {"name": "attend_step_16", "op": "attend", "seqs": 16, "heads": 16, "kv_heads": 8, "dim": 128, "rows": 1,
         "lo": 128, "hi": 32768, "type": "f16", "weights": True},
        # one stream far into a reading of three hours, wide groups of narrow heads
        {"name": "attend_step_131001", "op": "attend", "seqs": 1, "heads": 32, "kv_heads": 4, "dim": 64, "rows": 1,
         "lo": 131001, "hi": 131001, "type": "bf16", "weights": False},
        # the long-context prompt over its own rows
        {"name": "attend_prompt_2049", "op": "attend", "seqs": 1, "heads": 16, "kv_heads": 8, "dim": 128, "rows": 2049,
         "lo": 2049, "hi": 2049, "type": "f16", "weights": False},
        # three sessions resumed with 209 more rows (a voice clone's) behind long histories, weights kept
        {"name": "attend_resume_209", "op": "attend", "seqs": 3, "heads": 16, "kv_heads": 8, "dim": 128, "rows": 209,
         "lo": 4001, "hi": 12011, "type": "bf16", "weights": True},
        # one layer of one stream brought back to its bound, and read for a 16-bit cache
        {"name": "evict_2049", "op": "evict", "seqs": 1, "kv_heads": 8, "dim": 128, "lo": 2049, "hi": 2049,
         "keep": 1500, "sink": 4, "recent": 256},
        # the same for 16 long sessions at once
        {"name": "evict_16", "op": "evict", "seqs": 16, "kv_heads": 8, "dim": 128, "lo": 9000, "hi": 32768,
         "keep": 12001, "sink": 16, "recent": 4000},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend", "evict"])
    kv, group, dim = rng.choice([(8, 2, 128), (8, 2, 128), (4, 8, 64), (2, 4, 128), (16, 1, 64), (5, 3, 128), (1, 16, 128)])
    if op == "rope":
        return {"op": op, "tokens": _log(rng, 1, 12000), "heads": kv * group, "kv_heads": kv, "dim": dim,
                "rot": dim if rng.random() < 0.6 else 2 * rng.randrange(4, dim // 2), "from": rng.choice(["f32", "f16", "bf16"]),
                "to": rng.choice(["f16", "bf16"]), "inter": rng.random() < 0.4, "norm": rng.random() < 0.5,
                "factor": rng.choice([1.0, 1.0, 4.0, 32.0]), "far": _log(rng, 1, 1000000)}
    if op == "append":
        seqs = _log(rng, 1, 32)
        lo = rng.randrange(0, 3000)
        return {"op": op, "seqs": seqs, "kv_heads": kv, "dim": dim, "rows": _log(rng, 1, 2500 // seqs + 1), "lo": lo,
                "hi": lo + rng.randrange(0, 2000), "from": rng.choice(["f32", "f16", "bf16"])}
    if op == "evict":
        seqs = _log(rng, 1, 12)
        hi = _log(rng, 200, 24000)
        keep = max(24, int(hi * rng.uniform(0.3, 0.9)))
        return {"op": op, "seqs": seqs, "kv_heads": kv, "dim": dim, "lo": hi - rng.randrange(0, hi // 2), "hi": hi,
                "keep": keep, "sink": rng.randrange(0, 9), "recent": rng.randrange(1, keep // 2)}
    hi = _log(rng, 1, 100000)
    seqs = _log(rng, 1, max(1, min(16, 300000 // (hi * kv))))
    rows = rng.choice([1, 1, 1, rng.randrange(1, 9), _log(rng, 1, 1500)])
    rows = max(1, min(rows, hi, 60_000_000 // (hi * seqs * kv * group)))
    return {"op": op, "seqs": seqs, "heads": kv * group, "kv_heads": kv, "dim": dim, "rows": rows,
            "lo": max(rows, hi - rng.randrange(0, hi)), "hi": hi, "type": rng.choice(["f16", "bf16"]),
            "weights": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _lens(case):
    """Each sequence's length, spread evenly over the case's range in a mixed order, the ends among them."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    at = [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]
    return [at[(i * 7) % n] if n % 7 else at[i] for i in range(n)]


def _slots(n):
    return (n + 63) // 64 * 64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _inv_freq(rot, factor):
    """Frequencies of base 1e6 in 64 bits; a factor stretches the slow ones, keeps the fast ones (those with more
    than 32 turns in 32,768 positions) and blends between (one turn to 32)."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = 1e6 ** (-2.0 * i / rot)
    if factor != 1.0:
        turns = 32768 * f / (2 * math.pi)
        keep = ((turns.log() - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.cuda()


def _cache(case, g, lens, slots):
    """A cache whose first lens[s] slots hold N(0, 1) rows with a few wide dims, as normed keys have them."""
    s, h, d = case["seqs"], case["kv_heads"], case["dim"]
    wide = torch.ones(d, device="cuda")
    wide[3::29] = 4.0
    live = torch.arange(slots, device="cuda") < torch.tensor(lens, device="cuda")[:, None]
    c = {}
    for name in ("k", "v"):
        x = torch.randn(s, h, slots, d, generator=g, device="cuda") * (wide if name == "k" else 1.0)
        x *= live[:, None, :, None]
        x = x.view(s, h, slots // BLOCK, BLOCK * d)
        c[name + "s"] = x.abs().amax(-1) / 127.0
        x = torch.round(x / c[name + "s"].clamp_min(1e-30)[..., None])
        c[name] = x.view(s, h, slots, d).to(torch.int8)
    # a slot's drawn weight: heavy-tailed, as a few positions draw most of it
    c["acc"] = torch.exp(2.0 * torch.randn(s, h, slots, generator=g, device="cuda")) * 0.05 * live[:, None]
    return c


def _handle(c, weights=True):
    from qwen3_tts_amd import kv8
    return kv8.Cache(c["k"], c["v"], c["ks"], c["vs"], c["acc"] if weights else None)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "rope":
        t, d = case["tokens"], case["dim"]
        s["x"] = [torch.randn(t, n, d, generator=g, device="cuda").to(TYPES[case["from"]]) for n in (case["heads"], case["kv_heads"])]
        s["gain"] = [1 + 0.2 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None for _ in range(2)]
        s["pos"] = torch.arange(case["far"], case["far"] + t, device="cuda", dtype=torch.int32)
        s["inv_freq"] = _inv_freq(case["rot"], case["factor"])
        s["mscale"] = 0.1 * math.log(case["factor"]) + 1.0
        return s
    lens = _lens(case)
    s["lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
    slots = _slots(max(lens) + (case["rows"] if case["op"] == "append" else 0))
    s["cache"] = _cache(case, g, lens, slots)
    if case["op"] == "append":
        shape = (case["seqs"], case["rows"], case["kv_heads"], case["dim"])
        s["k"], s["v"] = (1.1 * torch.randn(shape, generator=g, device="cuda").to(TYPES[case["from"]]) for _ in range(2))
    elif case["op"] == "attend":
        s["q"] = (2.0 * torch.randn(case["seqs"], case["rows"], case["heads"], case["dim"], generator=g, device="cuda")).to(TYPES[case["type"]])
        s["scale"] = case["dim"] ** -0.5
    else:
        s["to"] = {k: torch.zeros_like(v[:, :, :_slots(case["keep"]) // (BLOCK if k in ("ks", "vs") else 1)]) for k, v in s["cache"].items()}
        s["first"] = torch.zeros_like(s["lens"])
    if own:
        # the views of the cache's memory that a program keeps
        s["handle"] = _handle(s["cache"], case.get("weights", True))
        if "to" in s:
            s["to_handle"] = _handle(s["to"])
    return s


# ---------------------------------------------------------------- the operators in elementary operations
def _rope(x, gain, pos, inv_freq, mscale, rot, inter, t):
    """x [tokens][heads][dim] normed (where it has a gain) and rotated, in type t; angles in 64 bits."""
    w = torch.float64 if t == torch.float64 else torch.float32
    z = x.to(w)
    if gain is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-6) * gain.to(w)
    a = pos.double()[:, None] * inv_freq
    c, s = (f(a).mul(mscale).to(w)[:, None] for f in (torch.cos, torch.sin))
    if inter:
        p, q = z[..., :rot:2], z[..., 1:rot:2]
        y = torch.stack((p * c - q * s, q * c + p * s), -1).flatten(-2)
    else:
        p, q = z[..., :rot // 2], z[..., rot // 2:rot]
        y = torch.cat((p * c - q * s, q * c + p * s), -1)
    return torch.cat((y, z[..., rot:]), -1).to(t)


def _append(c, name, x, start):
    """Rows x [S][n][H][D] quantised into the slots start[s] .. of c[name]."""
    s, n, h, d = x.shape
    blocks = (n + 2 * BLOCK - 2) // BLOCK
    codes, scales = c[name], c[name + "s"]
    at = start.long() // BLOCK * BLOCK                                          # the first block's first slot
    slot = at[:, None] + torch.arange(blocks * BLOCK, device=x.device)          # [S][window]
    row = slot - start[:, None]
    new = (row >= 0) & (row < n) & (slot < codes.shape[2])
    seq = torch.arange(s, device=x.device)[:, None]
    rows = torch.where(new[..., None, None], x[seq, row.clamp(0, n - 1)].float(), 0.0).transpose(1, 2)   # [S][H][window][D]
    held = slot.clamp(max=codes.shape[2] - 1)
    old = codes[seq, :, held].transpose(1, 2).float()
    blk = (at[:, None] // BLOCK + torch.arange(blocks, device=x.device)).clamp(max=scales.shape[2] - 1)
    s0 = scales[seq, :, blk].transpose(1, 2)                                    # [S][H][blocks]
    begun = (row < 0).view(s, blocks, BLOCK).any(-1)[:, None]
    s0 = torch.where(begun, s0, 0.0)
    s1 = torch.maximum(s0, rows.reshape(s, h, blocks, BLOCK * d).abs().amax(-1) / 127.0)
    ratio = torch.where(s1 > 0, s0 / s1, 1.0)
    wide = s1.repeat_interleave(BLOCK, -1)[..., None]
    q = torch.where(wide > 0, torch.round(rows / wide), 0.0)
    was = torch.where((row < 0)[:, None, :, None], torch.round(old * ratio.repeat_interleave(BLOCK, -1)[..., None]), old)
    q = torch.where(new[:, None, :, None], q, was).to(torch.int8)
    live = slot < codes.shape[2]
    codes[seq.expand_as(slot)[live], :, slot[live]] = q.transpose(1, 2)[live]
    touched = new.view(s, blocks, BLOCK).any(-1)
    scales[seq.expand_as(blk)[touched], :, blk[touched]] = s1.transpose(1, 2)[touched]
    if name == "k":
        c["acc"][seq.expand_as(slot)[new], :, slot[new]] = 0.0


def _values(c, name, first, n):
    """Slots first[s] .. + n of a cache as fp16 [S][n][H][D]; zeros past its end."""
    codes, scales = c[name], c[name + "s"]
    slot = first.long()[:, None] + torch.arange(n, device=codes.device)
    at = slot.clamp(max=codes.shape[2] - 1)
    seq = torch.arange(codes.shape[0], device=codes.device)[:, None]
    x = codes[seq, :, at].float() * scales[seq, :, at // BLOCK][..., None]
    return torch.where((slot < codes.shape[2])[..., None, None], x, 0.0).half()


def _attend(q, k, v, lens, scale, t):
    """q [S][n][Hq][D], k and v [S][H][C][D] in 32 (or 64) bits: (rows in type t, weights [S][H][C])."""
    s, n, hq, d = q.shape
    h, slots = k.shape[1], k.shape[2]
    w = k.dtype
    q = q.to(w).view(s, n, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(s, h, hq // h * n, d)
    x = torch.matmul(q, k.transpose(-1, -2)).view(s, h, hq // h, n, slots) * scale
    last = lens[:, None] - n + torch.arange(n, device=q.device)                 # [S][n]: the last slot of each row
    seen = torch.arange(slots, device=q.device) <= last[..., None]
    x = x.masked_fill(~seen[:, None, None], -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(x.view(s, h, -1, slots), v).view(s, h, hq // h, n, d).permute(0, 3, 1, 2, 4)
    return o.reshape(s, n, hq, d).to(t), x.sum((2, 3))


def _evict(c, to, lens, keep, sink, recent):
    """The kept slots of each (sequence, head), ascending (-1: none), and the cache compacted to them in `to`."""
    acc = c["acc"]
    slots = acc.shape[2]
    slot = torch.arange(slots, device=acc.device)
    n = lens.long()[:, None, None]
    left = n.clamp(max=keep)
    sure = (slot < sink) | (slot >= n - recent)
    key = torch.where(acc.isnan(), -torch.inf, acc) + 0.0
    # order: live before not, then those that stay in any case, then by weight, then by slot
    by = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.where(slot < n, torch.where(sure, 0, 1), 2).expand_as(acc).gather(-1, by)
    by = by.gather(-1, torch.sort(rank, dim=-1, stable=True).indices)[..., :keep]
    if by.shape[-1] < keep:
        by = torch.nn.functional.pad(by, (0, keep - by.shape[-1]))
    on = torch.arange(keep, device=acc.device) < left
    kept = torch.sort(torch.where(on, by, slots), -1).values
    at = torch.where(on, kept, 0)
    room = _slots(keep)
    pad = torch.nn.functional.pad
    for name in ("k", "v"):
        s0 = torch.where(on, c[name + "s"].gather(-1, at // BLOCK), 0.0)
        s1 = pad(s0, (0, room - keep)).view(*s0.shape[:2], room // BLOCK, BLOCK).amax(-1)
        wide = s1.repeat_interleave(BLOCK, -1)[..., :keep]
        ratio = torch.where(wide > 0, s0 / wide, 1.0)
        rows = c[name].gather(2, at[..., None].expand(*at.shape, c[name].shape[-1]))
        rows = torch.round(rows.float() * ratio[..., None]).to(torch.int8)
        to[name][:, :, :keep] = torch.where(on[..., None], rows, to[name][:, :, :keep])
        to[name + "s"][...] = torch.where(pad(on.expand(kept.shape), (0, room - keep)).view(*s1.shape, BLOCK).any(-1), s1, to[name + "s"])
    to["acc"][:, :, :keep] = torch.where(on, acc.gather(-1, at), to["acc"][:, :, :keep])
    return torch.where(on, kept, -1).int(), lens.clamp(max=keep)


def _plain(s):
    case, c = s["case"], s.get("cache")
    if case["op"] == "rope":
        return [_rope(x, g, s["pos"], s["inv_freq"], s["mscale"], case["rot"], case["inter"], TYPES[case["to"]])
                for x, g in zip(s["x"], s["gain"])]
    if case["op"] == "append":
        for name in ("k", "v"):
            _append(c, name, s[name], s["lens"])
        first, n = s["lens"] // BLOCK * BLOCK, case["rows"] + BLOCK - 1
        return {"k": _values(c, "k", first, n), "v": _values(c, "v", first, n), "ks": c["ks"], "vs": c["vs"], "acc": c["acc"]}
    if case["op"] == "attend":
        k, v = (c[n].float() * c[n + "s"].repeat_interleave(BLOCK, -1)[..., None] for n in ("k", "v"))
        o, w = _attend(s["q"], k, v, s["lens"], s["scale"], TYPES[case["type"]])
        if not case["weights"]:
            return o
        c["acc"] += w
        return {"out": o, "acc": c["acc"]}
    to = s["to"]
    kept, left = _evict(c, to, s["lens"], case["keep"], case["sink"], case["recent"])
    return {"kept": kept, "lens": left, "acc": to["acc"], "ks": to["ks"], "vs": to["vs"],
            "k": _values(to, "k", s["first"], case["keep"]), "v": _values(to, "v", s["first"], case["keep"])}


def run(s):
    if not own:
        return _plain(s)
    from qwen3_tts_amd import kv8
    case, c = s["case"], s.get("cache")
    if case["op"] == "rope":
        return kv8.rope(s["x"], s["pos"], s["inv_freq"], gains=s["gain"], eps=1e-6, mscale=s["mscale"],
                        interleaved=case["inter"], dtype=TYPES[case["to"]])
    if case["op"] == "append":
        kv8.append(s["handle"], s["k"], s["v"], s["lens"])
        k, v = kv8.read(s["handle"], s["lens"] // BLOCK * BLOCK, case["rows"] + BLOCK - 1, dtype=torch.float16)
        return {"k": k, "v": v, "ks": c["ks"], "vs": c["vs"], "acc": c["acc"]}
    if case["op"] == "attend":
        o = kv8.attend(s["handle"], s["q"], s["lens"], scale=s["scale"], weights=case["weights"])
        return {"out": o, "acc": c["acc"]} if case["weights"] else o
    to = s["to"]
    kept, left = kv8.evict(s["handle"], s["to_handle"], s["lens"], n_keep=case["keep"], n_sink=case["sink"],
                           n_recent=case["recent"])
    k, v = kv8.read(s["to_handle"], s["first"], case["keep"], dtype=torch.float16)
    return {"kept": kept, "lens": left, "acc": to["acc"], "ks": to["ks"], "vs": to["vs"], "k": k, "v": v}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    d, h = case["dim"], case["kv_heads"]
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + h) * d
        return {"bytes": n * (BYTES[case["from"]] + BYTES[case["to"]]), "flops": n * (7 if case["norm"] else 3)}
    lens = _lens(case)
    if case["op"] == "append":
        rows = case["seqs"] * case["rows"] * h * 2 * d
        back = case["seqs"] * (case["rows"] + BLOCK - 1) * h * 2 * d
        return {"bytes": rows * (BYTES[case["from"]] + 1) + back * (1 + 2), "flops": 4 * rows + back}
    if case["op"] == "attend":
        n, t = case["rows"], BYTES[case["type"]]
        io = case["seqs"] * n * case["heads"] * 2 * d * t
        pairs = sum(n * m - n * (n - 1) // 2 for m in lens) * case["heads"]
        slot = 2 * d + 8 / BLOCK + (8 if case["weights"] else 0)
        return {"bytes": io + sum(lens) * h * slot, "flops": pairs * 4 * d}
    left = sum(min(n, case["keep"]) for n in lens) * h
    return {"bytes": sum(lens) * h * 4 + left * (2 * 2 * d + 12) + left * 2 * d * (1 + 2), "flops": left * 2 * d * 2}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s.get("cache")
    if case["op"] == "rope":
        out = []
        half = case["rot"] // 2
        turn = torch.polar(torch.full_like(s["inv_freq"], s["mscale"]), torch.zeros_like(s["inv_freq"]))
        turn = turn * torch.exp(1j * (s["pos"].double()[:, None] * s["inv_freq"]))
        for x, gain in zip(s["x"], s["gain"]):
            x = x.double()
            if gain is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * gain.double()
            a = torch.arange(half, device=x.device)
            i, j = (2 * a, 2 * a + 1) if case["inter"] else (a, a + half)
            z = torch.complex(x[..., i], x[..., j]) * turn[:, None]
            y = x.clone()
            y[..., i], y[..., j] = z.real, z.imag
            out.append(y)
        return out
    lens = [int(n) for n in s["lens"]]
    if case["op"] == "attend":
        out, weight = [], c["acc"].double()
        n, hq = case["rows"], case["heads"]
        for b, m in enumerate(lens):
            k, v = (c[i][b].double() * c[i + "s"][b].double().repeat_interleave(BLOCK, -1)[..., None] for i in ("k", "v"))
            rows = torch.zeros(n, hq, case["dim"], dtype=torch.float64, device=k.device)
            last = m - n + torch.arange(n, device=k.device)
            for i in range(hq):
                g = i // (hq // case["kv_heads"])
                x = s["q"][b, :, i].double() @ k[g, :m].t() * s["scale"]
                x = torch.where(torch.arange(m, device=k.device) <= last[:, None], x, -torch.inf)
                p = torch.softmax(x, -1)
                rows[:, i] = p @ v[g, :m]
                weight[b, g, :m] += p.sum(0)
            out.append(rows)
        out = torch.stack(out)
        return {"out": out, "acc": weight} if case["weights"] else out
    if case["op"] == "append":
        out = {i: [] for i in ("k", "v")}
        scales = {i: c[i + "s"].double() for i in ("k", "v")}
        n = case["rows"]
        for b, m in enumerate(lens):
            first = m // BLOCK * BLOCK
            for name in ("k", "v"):
                x = torch.zeros(n + BLOCK - 1, case["kv_heads"], case["dim"], dtype=torch.float64, device=c["k"].device)
                for j in range(first, m + n, BLOCK):
                    new = s[name][b, max(j - m, 0):j + BLOCK - m].double()
                    held = c[name][b, :, j:m].double().transpose(0, 1) * (scales[name][b, :, j // BLOCK][:, None] if j < m else 0.0)
                    step = new.abs().amax((0, 2)) / 127
                    step = torch.maximum(step, scales[name][b, :, j // BLOCK]) if j < m else step
                    scales[name][b, :, j // BLOCK] = step
                    rows = torch.cat((held, new)) / step[:, None]
                    rows = torch.round(rows) * step[:, None]
                    x[j - first:j - first + rows.shape[0]] = rows
                out[name].append(x)
        acc = c["acc"].double()
        for b, m in enumerate(lens):
            acc[b, :, m:m + n] = 0
        return {"k": torch.stack(out["k"]), "v": torch.stack(out["v"]), "ks": scales["k"], "vs": scales["v"], "acc": acc}
    keep, room = case["keep"], _slots(case["keep"])
    res = {n: torch.zeros(case["seqs"], keep, case["kv_heads"], case["dim"], dtype=torch.float64, device="cuda") for n in ("k", "v")}
    res |= {n + "s": torch.zeros(case["seqs"], case["kv_heads"], room // BLOCK, dtype=torch.float64, device="cuda") for n in ("k", "v")}
    res["acc"] = torch.zeros(case["seqs"], case["kv_heads"], room, dtype=torch.float64, device="cuda")
    for b, m in enumerate(lens):
        for h in range(case["kv_heads"]):
            weight = c["acc"][b, h, :m].cpu().numpy()
            order = sorted(range(m), key=lambda t: (not (t < case["sink"] or t >= m - case["recent"]), -weight[t], t))
            at = torch.tensor(sorted(order[:keep]), device="cuda")
            res["acc"][b, h, :len(at)] = c["acc"][b, h, at].double()
            for name in ("k", "v"):
                s0 = c[name + "s"][b, h, at // BLOCK].double()
                step = torch.nn.functional.pad(s0, (0, room - len(at))).view(-1, BLOCK).amax(-1)
                mine = step.repeat_interleave(BLOCK)[:len(at)]
                x = torch.round(c[name][b, h, at].double() * (s0 / mine)[:, None]) * mine[:, None]
                res[name][b, :len(at), h], res[name + "s"][b, h] = x, step
    return {"kept": None, "lens": None, **res}
