"""Attention over so many keys that the tensor cores' sums, which round towards zero, would drift: sums, maxima that move, and
what is not finite, over more than 32768 keys, in every form of tile."""
import pytest
import torch

from adrastea_b200 import MatmulMask
from serving_oracle import assert_close, attend
from test_gpu_serving import gen, half, ints, view

pytestmark = pytest.mark.gpu
PAGE = 256
INF, NAN = float("inf"), float("nan")


def run(kernels, kind, q, k, v, scale, hint=None, spare=5):
    """One causal sequence: q [new, H, hd], k and v [n, Hk, hd], n a multiple of PAGE where `kind` is paged; `spare` rows of no
    sequence behind it are left alone."""
    new, H, hd = q.shape
    n, Hk = k.shape[:2]
    rows = torch.cat([q, q.new_full((spare, H, hd), NAN)])
    out = torch.full_like(rows, 3.0)
    if kind == "packed":
        k, v = (torch.cat([t, t.new_full((spare, Hk, hd), NAN)]) for t in (k, v))
        kernels.attention_packed(view(out), view(rows), view(k), view(v), ints([0, n]), hint or n, scale, MatmulMask.Causal)
    else:
        table = torch.arange(n // PAGE, dtype=torch.int32, device="cuda")[None].contiguous()
        pool = [t.view(n // PAGE, PAGE, Hk, hd) for t in (k, v)]
        kernels.attention_paged(view(out), view(rows), *pool, table, ints([0, new]), ints([n]), hint or new, scale,
                                kernels.attention_paged_workspace(H, Hk, hd))
    kernels.device_status()
    assert (out[new:] == 3.0).all()
    return out[:new]


# how it is called, new rows, positions, query heads, key heads, head_dim, max_q if not the rows
FAR = [("paged", 300, 1 << 19, 64, 1, 128, None), ("paged", 300, 1 << 19, 64, 1, 64, None),
       ("paged", 296, 1 << 21, 64, 1, 64, None), ("paged", 296, 1 << 21, 64, 1, 128, None),  # keys shared by two CTAs
       ("packed", 1 << 17, 1 << 17, 1, 1, 64, None), ("packed", 1 << 18, 1 << 18, 1, 1, 64, None),
       ("packed", 1 << 18, 1 << 18, 1, 1, 128, None)]


@pytest.mark.parametrize("kind,new,n,H,Hk,hd,hint", FAR)
def test_sums_over_many_keys_do_not_drift(kernels, kind, new, n, H, Hk, hd, hint):
    """Equal weights, which fp16 holds, and values of one sign: a mean.

    Bound: the output's rounding, 2^-11, and what is dropped within 32768 keys: 2048 sums of 16 products, which lose 2^-23 of
    what has been summed each."""
    g = gen(n + hd)
    q, k = torch.zeros((new, H, hd), dtype=torch.float16, device="cuda"), half(g, n, Hk, hd)
    v = (1 + torch.rand((n, Hk, hd), device="cuda", generator=g)).half()
    out = run(kernels, kind, q, k, v, 0.1, hint)
    for i in (0, 1, new // 3, new // 2, new - 2, new - 1):
        seen = n - new + i + 1
        want = v[:seen, 0].double().mean(0).expand(H, hd)
        assert_close(out[i], want, want * (2.0 ** -11 + 2.0 ** -12), i)


MOVES = [("paged", 300, 81920, 64, 1, 128, None), ("paged", 300, 81920, 64, 1, 64, None), ("paged", 298, 1 << 17, 64, 1, 64, None),
         ("paged", 148, 1 << 17, 128, 2, 128, None), ("paged", 148, 1 << 17, 128, 2, 64, None),
         ("packed", 70000, 70000, 2, 1, 64, None), ("packed", 70000, 70000, 4, 4, 64, None), ("packed", 70000, 70000, 2, 1, 128, None)]


def some_rows(new):
    return sorted({0, 1, new // 7, new // 2, new - 1} | {r for r in (8191, 8192, 8300, 12289, 32767, 32768, 33000, 66000) if r < new})


@pytest.mark.parametrize("kind,new,n,H,Hk,hd,hint", MOVES)
@pytest.mark.parametrize("shape", ["grow", "fall", "waves", "far", "minus"])
def test_maxima_that_move_over_many_keys(kernels, kind, new, n, H, Hk, hd, hint, shape):
    """Scores that grow by 60 over the keys (every part of the sum counts less and less), fall, rise and fall again; maxima of
    4 million; scores of -infinity up to the middle.  The oracle's bound, with 2^-12 of the weighted values' sizes for the sums
    (see above)."""
    g = gen(n + H)
    at = torch.linspace(0, 1, n, device="cuda")
    ramp = {"grow": 60 * at, "fall": -60 * at, "waves": 20 * torch.sin(at * 40) + 20 * at, "far": 60 * at,
            "minus": torch.where(at < 0.5, -INF, 10 * at)}[shape]
    q, k = 0.1 * half(g, new, H, hd), half(g, n, Hk, hd)
    q[..., 0], k[..., 0] = 1.0, ramp.half()[:, None]
    v = (0.5 + torch.rand((n, Hk, hd), device="cuda", generator=g)).half()
    scale = 1.0
    if shape == "far":   # every score of the ramp, a step of 512 apart
        q[..., 1:] = 0
        q[..., 0], k[..., 0] = 4096.0, (torch.floor(ramp * 16)).half()[:, None]
    out = run(kernels, kind, q, k, v, scale, hint)
    for i in some_rows(new):
        seen = n - new + i + 1
        first = int((at < 0.5).sum()) if shape == "minus" else 0   # (what is before has no weight)
        for h in {0, H - 1}:
            if seen <= first:
                assert out[i, h].isnan().all()
                continue
            kk, vv = k[first:seen, h // (H // Hk)][:, None], v[first:seen, h // (H // Hk)][:, None]
            want, tol = attend(q[i:i + 1, h:h + 1], kk, vv, scale, seen - first)
            assert_close(out[i:i + 1, h:h + 1], want, tol + want.abs() * 2.0 ** -12, (i, h))


@pytest.mark.parametrize("kind,new,n,H,Hk,hd,hint", MOVES)
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_bad_value_among_many(kernels, kind, new, n, H, Hk, hd, hint, value):
    """One token's value is not finite in one column: the rows before it, and the other columns, do not see it."""
    for at in {100, n - new // 2, n - 1} if kind == "packed" else {100, n // 2, n - new // 2}:
        g = gen(n + H + at)
        q, k = half(g, new, H, hd), half(g, n, Hk, hd)
        v = (0.5 + torch.rand((n, Hk, hd), device="cuda", generator=g)).half()
        clean = run(kernels, kind, q, k, v, 0.1, hint)
        v[at, :, 3] = value
        out = run(kernels, kind, q, k, v, 0.1, hint)
        first = max(0, at - (n - new))
        # (rows that share a block with it may be summed in another order: 2^-22 of the 128 weights and more; fp16 rounds both)
        same = torch.isclose(out.float(), clean.float(), rtol=2.0 ** -10, atol=2.0 ** -14)
        assert same[:first].all(), at
        assert same[..., 4:].all() and same[..., :3].all(), at
        assert not out[first:, :, 3].isfinite().any(), at


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk", [(2, 2), (64, 1)])
def test_more_rows_than_positions(kernels, hd, H, Hk):
    """The first rows lie before position 0 and are zeros, in a sequence of many positions all the same."""
    new, n = 50000, 40000
    g = gen(hd + H)
    q, k, v = half(g, new, H, hd), half(g, n, Hk, hd), half(g, n, Hk, hd)
    out = torch.full_like(q, NAN)
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda")[None].contiguous()
    kernels.attention_paged(view(out), view(q), k.view(n // 64, 64, Hk, hd), v.view(n // 64, 64, Hk, hd), table, ints([0, new]),
                            ints([n]), new, 0.1, kernels.attention_paged_workspace(H, Hk, hd))
    kernels.device_status()
    assert not out[:new - n].any()
    for i in (new - n, new - n + 1, new - 3000, new - 1):
        seen = n - new + i + 1
        want, tol = attend(q[i:i + 1, :1], k[:seen, :1], v[:seen, :1], 0.1, seen)
        assert_close(out[i:i + 1, :1], want, tol + 2.0 ** -12, i)


# ------------------------------------------------------------------ a few rows
# sequences, new rows, positions, query heads, key heads, head_dim: whole sequences to a CTA
FEW = [(40, 1, 1 << 20, 8, 8, 64), (40, 1, 1 << 20, 8, 8, 128), (40, 1, 1 << 20, 64, 8, 64), (20, 1, 1 << 20, 128, 8, 128),
       (40, 5, 1 << 20, 32, 8, 128), (40, 20, 1 << 20, 8, 8, 64), (3, 1, 1 << 20, 4, 2, 128)]


def few(kernels, q, k, v, S, scale, new):
    """`S` sequences that share all their pages."""
    n, Hk, hd = k.shape
    H = q.shape[1]
    table = torch.arange(n // PAGE, dtype=torch.int32, device="cuda")[None].expand(S, -1).contiguous()
    pool = [t.view(n // PAGE, PAGE, Hk, hd) for t in (k, v)]
    out = torch.full((S * new + 3, H, hd), 3.0, dtype=torch.float16, device="cuda")
    rows = torch.cat([q, q.new_full((3, H, hd), NAN)])
    kernels.attention_paged(view(out), view(rows), *pool, table, ints([i * new for i in range(S + 1)]), ints([n] * S), new, scale,
                            kernels.attention_paged_workspace(H, Hk, hd))
    kernels.device_status()
    assert (out[S * new:] == 3.0).all()
    return out[:S * new]


@pytest.mark.parametrize("S,new,n,H,Hk,hd", FEW)
def test_sums_of_few_rows_do_not_drift(kernels, S, new, n, H, Hk, hd):
    """As above, with 32768 keys to a warp between two beginnings."""
    g = gen(n + hd)
    q, k = torch.zeros((S * new, H, hd), dtype=torch.float16, device="cuda"), half(g, n, Hk, hd)
    v = (1 + torch.rand((n, Hk, hd), device="cuda", generator=g)).half()
    out = few(kernels, q, k, v, S, 0.1, new)
    want = v.double().mean(0).repeat_interleave(H // Hk, 0)
    # (an earlier row sees up to 19 keys fewer of a million, whose mean differs by less than 2^-15)
    assert_close(out, want.expand(S * new, H, hd), (want * (2.0 ** -11 + 2.0 ** -12) + 2.0 ** -15).expand(S * new, H, hd))


@pytest.mark.parametrize("S,new,n,H,Hk,hd", FEW)
@pytest.mark.parametrize("shape", ["grow", "fall", "waves", "minus", "nan", "inf"])
def test_maxima_of_few_rows_that_move(kernels, S, new, n, H, Hk, hd, shape):
    """Scores that grow over the keys, fall, rise and fall again; that are -infinity up to the middle; a value that is not
    finite, which every row sees: other columns do not."""
    n = 300 * 1024
    g = gen(n + H)
    at = torch.linspace(0, 1, n, device="cuda")
    ramp = {"grow": 40 * at, "fall": -40 * at, "waves": 15 * torch.sin(at * 40) + 15 * at,
            "minus": torch.where(at < 0.5, -INF, 10 * at)}.get(shape, 0 * at)
    q, k = 0.1 * half(g, S * new, H, hd), half(g, n, Hk, hd)
    q[..., 0], k[..., 0] = 1.0, ramp.half()[:, None]
    v = (0.5 + torch.rand((n, Hk, hd), device="cuda", generator=g)).half()
    first = int((at < 0.5).sum()) if shape == "minus" else 0
    clean = v.clone()
    if shape in ("nan", "inf"):
        v[1000, :, 3] = NAN if shape == "nan" else INF
    out = few(kernels, q, k, v, S, 1.0, new)
    if shape in ("nan", "inf"):
        assert not out[..., 3].isfinite().any()
        out[..., 3] = 0
        clean[..., 3] = 0
    for i in sorted({0, new - 1, S * new // 2, S * new - 1}):
        seen = n - new + i % new + 1
        for h in {0, H - 1}:
            kk, vv = k[first:seen, h // (H // Hk)][:, None], clean[first:seen, h // (H // Hk)][:, None]
            want, tol = attend(q[i:i + 1, h:h + 1], kk, vv, 1.0, seen - first)
            assert_close(out[i:i + 1, h:h + 1], want, tol + want.abs() * 2.0 ** -12, (i, h))


# ------------------------------------------------------------------ long and short ones together
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk", [(4, 2), (16, 16)])
def test_long_and_short_prompts_together(kernels, hd, causal, H, Hk):
    lens = [5, 70000, 300, 0, 40000, 129]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    g = gen(hd + H)
    q, k = half(g, cu[-1] + 4, H, hd), half(g, cu[-1] + 4, Hk, hd)
    v = (0.5 + torch.rand((cu[-1] + 4, Hk, hd), device="cuda", generator=g)).half()
    for t in (q, k, v):
        t[cu[-1]:] = NAN
    out = torch.full_like(q, 3.0)
    kernels.attention_packed(view(out), view(q), view(k), view(v), ints(cu), max(lens), 0.1,
                             MatmulMask.Causal if causal else MatmulMask.None_)
    kernels.device_status()
    assert (out[cu[-1]:] == 3.0).all()
    for s, n in enumerate(lens):
        for i in sorted({0, n // 3, n - 1} | {r for r in (32767, 32768, 65600) if r < n}) if n else ():
            for h in (0, H - 1):
                seen = i + 1 if causal else n
                rows, kh = slice(cu[s], cu[s] + seen), slice(h // (H // Hk), h // (H // Hk) + 1)
                at = slice(cu[s] + i, cu[s] + i + 1)
                want, tol = attend(q[at, h:h + 1], k[rows, kh], v[rows, kh], 0.1, seen)
                assert_close(out[at, h:h + 1], want, tol + want.abs() * 2.0 ** -12, (s, i, h))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk", [(8, 2), (64, 32)])
@pytest.mark.parametrize("new,lens", [([300, 1, 40, 90], [100000, 120000, 50, 33000]), ([200] * 4, [90000, 200, 70000, 1000])])
def test_chunks_and_tokens_over_long_and_short_caches(kernels, hd, H, Hk, new, lens):
    g = gen(hd + H + new[1])
    need = [-(-n // PAGE) for n in lens]
    cu, first = [0], [0]
    for m, pages in zip(new, need):
        cu.append(cu[-1] + m)
        first.append(first[-1] + pages)
    pool_k = half(g, first[-1], PAGE, Hk, hd)
    pool_v = (0.5 + torch.rand((first[-1], PAGE, Hk, hd), device="cuda", generator=g)).half()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    for s, m in enumerate(need):
        table[s, :m] = torch.arange(first[s], first[s + 1], device="cuda")
    q = half(g, cu[-1], H, hd)
    out, ws = torch.full_like(q, NAN), kernels.attention_paged_workspace(H, Hk, hd)
    for _ in range(2):
        kernels.attention_paged(view(out), view(q), pool_k, pool_v, table, ints(cu), ints(lens), max(new), 0.1, ws)
    kernels.device_status()
    for s, (m, n) in enumerate(zip(new, lens)):
        keys, values = (t[first[s]:first[s + 1]].flatten(0, 1) for t in (pool_k, pool_v))
        for i in sorted({0, m // 2, m - 1}):
            for h in (0, H - 1):
                seen, kh = n - m + i + 1, slice(h // (H // Hk), h // (H // Hk) + 1)
                at = slice(cu[s] + i, cu[s] + i + 1)
                want, tol = attend(q[at, h:h + 1], keys[:seen, kh], values[:seen, kh], 0.1, seen)
                assert_close(out[at, h:h + 1], want, tol + want.abs() * 2.0 ** -12, (s, i, h))
