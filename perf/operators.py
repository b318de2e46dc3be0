"""The operators of serving requests of different lengths, as measurable cases.

Kinds of case:

  rope      rotation of packed rows (q and k of a projection side by side) at given positions:
            pairs (2i, 2i+1) or (i, i + d/2), all or part of the head, frequencies plain or scaled
            for long contexts (`GpuKernels.rope_f16`)
  append    q and k of new tokens rotated, k and v written to the pages of their sequences
            (`GpuKernels.rope_append_paged`)
  packed    attention of whole prompts of different lengths that lie one behind the other, causal or
            unmasked, several query heads to a key head (`GpuKernels.attention_packed`)
  paged     attention of one or more new tokens per sequence over a paged cache
            (`GpuKernels.attention_paged`)

`run` computes them in elementary torch operations in 32 bits (angles in 64), or, with `own` set,
through the library's entry points.
"""
from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

own = False

THETA = 10000.0
NO_SCALING = dict(scaling="none", factor=1.0, original=0)


def listed():
    return [
        # q and k of a decode step of sixteen users of the 7B shape, rotated where the projection left them
        dict(name="rope_decode_16x64", kind="rope", tokens=16, heads=64, head_dim=128, rotary=128,
             layout="interleaved", pos0=575, **NO_SCALING),
        # a prompt that continues a long document: half layout on half of the head, far positions
        dict(name="rope_4111x40_half_far", kind="rope", tokens=4111, heads=40, head_dim=128, rotary=64,
             layout="half", pos0=126000, scaling="yarn", factor=16.0, original=8192),
        # the decode step's append: one token for each of sixteen users, heads of the 7B shape
        dict(name="append_decode_16", kind="append", seqs=16, shortest=17, longest=640, new_min=1, new_max=1,
             heads=32, kv_heads=32, head_dim=128, page=16, rotary=128, layout="interleaved", mix=1, **NO_SCALING),
        # five prompts that enter the cache together, four query heads to a key head
        dict(name="append_prompts_5", kind="append", seqs=5, shortest=700, longest=4096, new_min=700, new_max=4096,
             heads=32, kv_heads=8, head_dim=128, page=64, rotary=128, layout="half", mix=2, scaling="bands",
             factor=8.0, original=8192),
        # short texts, one of them of a single token
        dict(name="packed_texts_7x77_hd64", kind="packed", seqs=7, shortest=1, longest=77, heads=16, kv_heads=16,
             head_dim=64, causal=True, fused=False, mix=3),
        # images of the encoder, all of 257 tokens, every token sees every other
        dict(name="packed_images_32x257_hd64", kind="packed", seqs=32, shortest=257, longest=257, heads=16,
             kv_heads=16, head_dim=64, causal=False, fused=False, mix=4),
        # sixteen prompts of the 7B shape
        dict(name="packed_prompts_16x512", kind="packed", seqs=16, shortest=64, longest=512, heads=32, kv_heads=32,
             head_dim=128, causal=True, fused=True, mix=5),
        # two long documents, eight query heads to a key head
        dict(name="packed_long_2x8192", kind="packed", seqs=2, shortest=8191, longest=8192, heads=64, kv_heads=8,
             head_dim=128, causal=True, fused=True, mix=6),
        # the next token of one user in the middle of a conversation
        dict(name="paged_decode_1x600", kind="paged", seqs=1, shortest=600, longest=600, new_min=1, new_max=1,
             heads=32, kv_heads=32, head_dim=128, page=16, mix=7),
        # the next tokens of many users with contexts of very different lengths
        dict(name="paged_decode_64x8192", kind="paged", seqs=64, shortest=128, longest=8192, new_min=1, new_max=1,
             heads=32, kv_heads=8, head_dim=128, page=16, mix=8),
        # the next token over one very long document
        dict(name="paged_decode_1x131072", kind="paged", seqs=1, shortest=131072, longest=131072, new_min=1,
             new_max=1, heads=64, kv_heads=8, head_dim=128, page=64, mix=9),
        # chunks of prompts that are taken in piece by piece behind what is cached already
        dict(name="paged_chunks_4x512", kind="paged", seqs=4, shortest=2000, longest=16384, new_min=512, new_max=512,
             heads=32, kv_heads=8, head_dim=128, page=32, mix=10),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(32, 32), (32, 8), (64, 8), (16, 16), (20, 4), (14, 2), (40, 40), (8, 1)]


def _draw_rotation(rng, head_dim):
    scaling = rng.choice(["none", "linear", "base", "bands", "yarn"])
    rotary = head_dim if rng.random() < 0.6 else 2 * rng.randint(4, head_dim // 2)
    return dict(rotary=rotary, layout=rng.choice(["interleaved", "half"]), scaling=scaling,
                factor=1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 16])),
                original=0 if scaling in ("none", "linear", "base") else rng.choice([2048, 4096, 8192]))


def draw(rng):
    kind = rng.choice(["rope", "append", "packed", "packed", "paged", "paged", "paged"])
    head_dim = rng.choice([64, 128, 128])
    heads, kv_heads = rng.choice(HEADS)
    mix = rng.randrange(1 << 30)
    if kind == "rope":
        return dict(kind=kind, tokens=_log(rng, 1, 8192), heads=heads + kv_heads, head_dim=head_dim,
                    pos0=_log(rng, 1, 1 << 20), **_draw_rotation(rng, head_dim))
    if kind == "append":
        new_max = _log(rng, 1, 4096)
        seqs = _log(rng, 1, max(1, min(256, 8192 // new_max)))
        longest = _log(rng, new_max, max(new_max, (1 << 19) // (kv_heads * seqs)))
        return dict(kind=kind, seqs=seqs, shortest=rng.randint(1, longest), longest=longest, new_min=1,
                    new_max=new_max, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    page=rng.choice([16, 32, 64, 128, 256]), mix=mix, **_draw_rotation(rng, head_dim))
    if kind == "packed":
        longest = _log(rng, 8, 8192)
        seqs = _log(rng, 1, max(1, min(128, 16384 // longest)))
        return dict(kind=kind, seqs=seqs, shortest=rng.randint(1, longest), longest=longest, heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, causal=rng.random() < 0.8, fused=rng.random() < 0.7, mix=mix)
    # decode, a few tokens at a time, or chunks
    new_max = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1024)])
    most = min(524288, (1 << 22) // kv_heads) if new_max < 9 else 32768  # positions of all sequences
    longest = _log(rng, max(16, new_max), min(131072, most) if new_max < 9 else 16384)
    seqs = _log(rng, 1, max(1, min(128, most // longest, 2048 // new_max)))
    return dict(kind=kind, seqs=seqs, shortest=rng.randint(1, longest), longest=longest,
                new_min=1 if rng.random() < 0.5 else new_max, new_max=new_max, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=rng.choice([16, 32, 64, 128, 256]), mix=mix)


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """(new tokens, positions with them) of every sequence; one of them has the longest of both."""
    rng = random.Random(case["mix"])
    lens = [_log(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lens[rng.randrange(case["seqs"])] = case["longest"]
    if case["kind"] == "packed":
        return lens, lens
    if case["new_min"] == case["new_max"] == 1:
        return [1] * len(lens), lens
    if (case["new_min"], case["new_max"]) == (case["shortest"], case["longest"]):
        return lens, lens  # whole prompts
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in lens]
    return [min(a, b) for a, b in zip(new, lens)], lens


def work(case):
    hd = case["head_dim"]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * hd
        turned = case["tokens"] * case["heads"] * case["rotary"]
        return {"bytes": 4 * n + 4 * case["tokens"], "flops": 3 * turned}
    new, lens = _lengths(case)
    H, Hk = case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        per_token = 4 * hd * (H + 2 * Hk)  # read and written once
        pages = sum((n - 1) // case["page"] - (n - m) // case["page"] + 1 for m, n in zip(new, lens))
        return {"bytes": per_token * sum(new) + 4 * (pages + 2 * len(lens) + 1),
                "flops": 3 * case["rotary"] * (H + Hk) * sum(new)}
    if case["kind"] == "packed":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": 2 * hd * (2 * H + 2 * Hk) * sum(lens) + 4 * (len(lens) + 1), "flops": 4 * hd * H * pairs}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(new, lens))
    pages = sum(-(-n // case["page"]) for n in lens)
    return {"bytes": 2 * hd * (2 * H * sum(new) + 2 * Hk * sum(lens)) + 4 * (pages + 2 * len(lens) + 1),
            "flops": 4 * hd * H * pairs}


# ------------------------------------------------------------------ inputs
@functools.lru_cache(maxsize=None)
def _kernels():
    """The library's handle, opened once, with early launch on as a serving program sets it."""
    from adrastea_b200 import GpuKernels
    k = GpuKernels()
    k.set_tunable("pdl", 1)
    return k


def _rope_table(case):
    from adrastea_b200 import RopeLayout, RopeScaling
    scaling = {"none": lambda: RopeScaling.Identity(), "linear": lambda: RopeScaling.Linear(case["factor"]),
               "base": lambda: RopeScaling.Base(case["factor"]),
               "bands": lambda: RopeScaling.Bands(case["factor"], case["original"], 1.0, 4.0),
               "yarn": lambda: RopeScaling.Yarn(case["factor"], case["original"], 32.0, 1.0)}[case["scaling"]]()
    layout = RopeLayout.Half if case["layout"] == "half" else RopeLayout.Interleaved
    return _kernels().rope_table(case["rotary"], THETA, layout, scaling)


def _pages(case, lens, gen):
    """A block table over a pool of shuffled pages, a few of them unused; -1 behind a sequence's last page."""
    need = [-(-n // case["page"]) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    half = lambda *s: torch.randn(s, device="cuda", generator=gen).half()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    hd = case["head_dim"]
    st = dict(case=case)
    if case["kind"] == "rope":
        T, H = case["tokens"], case["heads"]
        # the rows hold v behind q and k: the rotated part is a view with a wider pitch
        st["rows"] = half(T, (H + 8) * hd)
        st["x"] = st["rows"].view(T, H + 8, hd)[:, :H]
        st["positions"] = ints(case["pos0"]) + torch.randperm(T, generator=gen, device="cuda").to(torch.int32)
        st["out"] = torch.zeros((T, H, hd), dtype=torch.float16, device="cuda")
        if own:
            st["table"] = _rope_table(case)
        return st
    new, lens = _lengths(case)
    H, Hk, T = case["heads"], case["kv_heads"], sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    st.update(new=new, lens=lens, cu=cu, cu_q=ints(cu), kv_len=ints(lens))
    if case["kind"] == "append":
        st["qkv"] = half(T, (H + 2 * Hk) * hd).view(T, H + 2 * Hk, hd)
        st["block_table"], pool = _pages(case, lens, gen)
        st["k_pages"] = torch.zeros((pool, case["page"], Hk, hd), dtype=torch.float16, device="cuda")
        st["v_pages"] = torch.zeros_like(st["k_pages"])
        st["q_out"] = torch.zeros((T, H, hd), dtype=torch.float16, device="cuda")
        if own:
            st["table"] = _rope_table(case)
        return st
    st["scale"] = 1.0 / math.sqrt(hd)
    st["out"] = torch.zeros((T, H, hd), dtype=torch.float16, device="cuda")
    if case["kind"] == "packed":
        # q, k and v side by side in the rows of one projection, or tensors of their own
        heads = [H, Hk, Hk]
        st["q"], st["k"], st["v"] = (half(T, sum(heads), hd).split(heads, 1) if case["fused"] else
                                     [half(T, n, hd) for n in heads])
        return st
    st["q"] = half(T, H, hd)
    st["block_table"], pool = _pages(case, lens, gen)
    st["k_pages"] = half(pool, case["page"], Hk, hd)
    st["v_pages"] = half(pool, case["page"], Hk, hd)
    if own:
        st["workspace"] = _kernels().attention_paged_workspace(H, Hk, hd)
    return st


# ------------------------------------------------------------------ one pass
def _own(st):
    from adrastea_b200 import MatmulMask, TensorView
    k, case, view = _kernels(), st["case"], TensorView.of
    if case["kind"] == "rope":
        k.rope_f16(view(st["out"]), view(st["x"]), st["positions"], st["table"])
        return st["out"]
    H, Hk = case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        q, key, val = (view(t) for t in st["qkv"].split([H, Hk, Hk], 1))
        k.rope_append_paged(view(st["q_out"]), q, key, val, st["k_pages"], st["v_pages"], st["block_table"],
                            st["cu_q"], st["kv_len"], st["table"])
        return [st["q_out"], st["k_pages"], st["v_pages"]]
    if case["kind"] == "packed":
        k.attention_packed(view(st["out"]), view(st["q"]), view(st["k"]), view(st["v"]), st["cu_q"],
                           max(st["lens"]), st["scale"],
                           MatmulMask.Causal if case["causal"] else MatmulMask.None_)
        return st["out"]
    k.attention_paged(view(st["out"]), view(st["q"]), st["k_pages"], st["v_pages"], st["block_table"], st["cu_q"],
                      st["kv_len"], max(st["new"]), st["scale"], st["workspace"])
    return st["out"]


def _frequencies(case):
    """Angle per position of every pair, in 64 bits, and what the rotated pair is multiplied by."""
    d, s, theta = case["rotary"], case["factor"], THETA
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "base":
        theta = theta * s ** (d / (d - 2))
    f = torch.exp(-2.0 * i / d * math.log(theta))
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "bands":
        turns = case["original"] * f / (2 * math.pi)  # of the original context
        blend = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f / s * (1 - blend) + f * blend
    if case["scaling"] == "yarn":
        at = lambda turns: d * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f / s * ramp + f * (1 - ramp)
    return f, 0.1 * math.log(s) + 1.0 if case["scaling"] == "yarn" else 1.0


def _rotate(case, x, positions):
    """x [T, H, hd] fp16 at positions [T]: rotated in 32 bits, rounded once."""
    d = case["rotary"]
    f, amplitude = _frequencies(case)
    angle = positions.double()[:, None] * f
    c, s = (amplitude * angle.cos()).float()[:, None], (amplitude * angle.sin()).float()[:, None]
    y = x.float().clone()
    if case["layout"] == "half":
        a, b = y[..., :d // 2].clone(), y[..., d // 2:d].clone()
        y[..., :d // 2], y[..., d // 2:d] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., 0:d:2].clone(), y[..., 1:d:2].clone()
        y[..., 0:d:2], y[..., 1:d:2] = a * c - b * s, b * c + a * s
    return y.half()


def _attend(out, q, k, v, scale, first):
    """q [m, H, hd], k and v [n, Hk, hd]: row i sees the first `first + i` keys (all of them where None)."""
    m, H, hd = q.shape
    n, Hk = k.shape[:2]
    g = H // Hk
    step = max(1, (1 << 30) // (g * m * n))  # key heads at a time: a few GB of scores
    for h in range(0, Hk, step):
        e = min(Hk, h + step)
        qh = q[:, h * g:e * g].float().unflatten(1, (e - h, g)).permute(1, 2, 0, 3)   # [heads, g, m, hd]
        kh, vh = (t[:, h:e].float().permute(1, 0, 2).unsqueeze(1) for t in (k, v))    # [heads, 1, n, hd]
        s = torch.matmul(qh, kh.transpose(-1, -2)) * scale
        if first is not None:
            seen = torch.arange(n, device=q.device)[None] < first + torch.arange(m, device=q.device)[:, None]
            s = s.masked_fill(~seen, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, vh) / p.sum(-1, keepdim=True)
        out[:, h * g:e * g] = o.permute(2, 0, 1, 3).flatten(1, 2).half()


def _gather(pages, table, n):
    """The first n positions of one sequence, [n, Hk, hd]."""
    return pages[table[:-(-n // pages.shape[1])].long()].flatten(0, 1)[:n]


def run(st):
    if own:
        return _own(st)
    case = st["case"]
    if case["kind"] == "rope":
        st["out"].copy_(_rotate(case, st["x"], st["positions"]))
        return st["out"]
    H, Hk = case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        q, key, val = st["qkv"].split([H, Hk, Hk], 1)
        seq = torch.repeat_interleave(torch.arange(len(st["new"]), device="cuda"), st["cu_q"].diff(),
                                      output_size=q.shape[0])
        at = torch.arange(q.shape[0], device="cuda") - st["cu_q"][seq + 1] + st["kv_len"][seq]
        st["q_out"].copy_(_rotate(case, q, at))
        page, slot = st["block_table"][seq, at // case["page"]].long(), at % case["page"]
        st["k_pages"][page, slot] = _rotate(case, key, at)
        st["v_pages"][page, slot] = val
        return [st["q_out"], st["k_pages"], st["v_pages"]]
    for s, (m, n) in enumerate(zip(st["new"], st["lens"])):
        rows = slice(st["cu"][s], st["cu"][s + 1])
        if case["kind"] == "packed":
            _attend(st["out"][rows], st["q"][rows], st["k"][rows], st["v"][rows], st["scale"],
                    1 if case["causal"] else None)
        else:
            k, v = (_gather(st[p], st["block_table"][s], n) for p in ("k_pages", "v_pages"))
            _attend(st["out"][rows], st["q"][rows], k, v, st["scale"], n - m + 1)
    return st["out"]


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_turns(case):
    """Pair by pair from the definition of each scaling: (angle per position, amplitude)."""
    d, s, L = case["rotary"], case["factor"], case["original"]
    kind, out = case["scaling"], []
    for i in range(d // 2):
        f = THETA ** (-2.0 * i / d)
        if kind == "linear":
            f /= s
        elif kind == "base":
            f = (THETA * s ** (d / (d - 2.0))) ** (-2.0 * i / d)
        elif kind == "bands":
            wave = 2.0 * math.pi / f
            if wave > L:                 # less than one turn: stretched
                f /= s
            elif wave >= L / 4.0:        # between: blended
                w = (L / wave - 1.0) / 3.0
                f = (1.0 - w) * f / s + w * f
        elif kind == "yarn":
            edge = [d * math.log(L / (b * 2.0 * math.pi)) / (2.0 * math.log(THETA)) for b in (32.0, 1.0)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), d - 1)
            w = min(1.0, max(0.0, (i - lo) / (hi - lo if hi > lo else 0.001)))
            f = w * (f / s) + (1.0 - w) * f
        out.append(f)
    return np.array(out), (1.0 + 0.1 * math.log(s)) if kind == "yarn" else 1.0


def _exact_rotation(case, x, positions):
    """Each pair as a complex number times amplitude * e^(i angle)."""
    d = case["rotary"]
    f, amplitude = _exact_turns(case)
    angle = torch.outer(positions.to(torch.float64), torch.from_numpy(f).to(x.device))
    turn = torch.polar(torch.full_like(angle, amplitude), angle).unsqueeze(1)
    x = x.to(torch.float64)
    if case["layout"] == "half":
        z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:d].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(x[..., :d].unflatten(-1, (d // 2, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat([head, x[..., d:]], -1)


def _exact_attention(q, k, v, scale, behind):
    """q [m, H, hd] over k, v [n, Hk, hd] in 64 bits, some query rows at a time; row i sees the keys up to `behind + i`."""
    m, H, hd = q.shape
    n, Hk = k.shape[:2]
    K, V = k.double().permute(1, 2, 0), v.double().permute(1, 0, 2)             # [Hk, hd, n], [Hk, n, hd]
    out = torch.empty((m, H, hd), dtype=torch.float64, device=q.device)
    step = max(1, min(m, (1 << 28) // (H * n)))
    at = torch.arange(n, device=q.device)
    for lo in range(0, m, step):
        hi = min(m, lo + step)
        rows = q[lo:hi].double().unflatten(1, (Hk, H // Hk)).permute(1, 2, 0, 3).flatten(1, 2)   # [Hk, g * rows, hd]
        s = torch.bmm(rows, K).mul_(scale).unflatten(1, (H // Hk, hi - lo))
        if behind is not None:
            s.masked_fill_(at > behind + torch.arange(lo, hi, device=q.device).unsqueeze(1), float("-inf"))
        w = torch.softmax(s, -1).flatten(1, 2)
        out[lo:hi] = torch.bmm(w, V).unflatten(1, (H // Hk, hi - lo)).permute(2, 0, 1, 3).flatten(1, 2)
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    if case["kind"] == "rope":
        return _exact_rotation(case, st["x"], st["positions"])
    H, Hk = case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        q, key, val = st["qkv"].split([H, Hk, Hk], 1)
        at = torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(st["new"], st["lens"])])
        k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
        turned = _exact_rotation(case, key, at)
        table = st["block_table"].cpu().numpy()
        pages = np.concatenate([table[s][np.arange(n - m, n) // case["page"]]
                                for s, (m, n) in enumerate(zip(st["new"], st["lens"]))])
        pages = torch.from_numpy(pages.astype(np.int64)).cuda()
        k_pages[pages, at % case["page"]] = turned
        v_pages[pages, at % case["page"]] = val.double()
        return [_exact_rotation(case, q, at), k_pages, v_pages]
    out = torch.empty(st["out"].shape, dtype=torch.float64, device="cuda")
    for s, (m, n) in enumerate(zip(st["new"], st["lens"])):
        lo, hi = st["cu"][s], st["cu"][s + 1]
        if case["kind"] == "packed":
            out[lo:hi] = _exact_attention(st["q"][lo:hi], st["k"][lo:hi], st["v"][lo:hi], st["scale"],
                                          0 if case["causal"] else None)
        else:
            idx = st["block_table"][s, :-(-n // case["page"])].long()
            k, v = (st[p].index_select(0, idx).reshape(-1, Hk, case["head_dim"])[:n] for p in ("k_pages", "v_pages"))
            out[lo:hi] = _exact_attention(st["q"][lo:hi], k, v, st["scale"], n - m)
    return out
