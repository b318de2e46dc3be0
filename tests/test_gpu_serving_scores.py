"""Scores where the attention over sequences of different lengths can lose a row: weights far below the largest one, scores
of many millions, scores that are not finite.  Every form of every kernel, against 64-bit forms."""
import math

import pytest
import torch

from adrastea_b200 import MatmulMask
from serving_oracle import assert_close
from test_gpu_serving import Pages, gen, half, ints, view

pytestmark = pytest.mark.gpu
INF = float("inf")

# how it is called, new rows, positions, query heads, key heads, head_dim
FORMS = [("paged", 1, 900, 8, 2, 64), ("paged", 1, 900, 8, 2, 128), ("paged", 1, 9000, 8, 1, 128),  # one row tile, many parts
         ("paged", 7, 900, 4, 1, 64), ("paged", 7, 900, 4, 1, 128),                                 # 28 rows
         ("paged", 300, 900, 64, 64, 64), ("paged", 90, 400, 32, 32, 128), ("paged", 300, 900, 64, 64, 128),  # tiles
         ("paged", 90, 900, 32, 32, 64), ("paged", 300, 900, 32, 32, 128),                          # keys shared out
         ("paged", 90, 5000, 4, 1, 64), ("paged", 90, 5000, 4, 1, 128),
         ("packed", 300, 300, 8, 1, 64), ("packed", 300, 300, 8, 1, 128),
         ("packed", 300, 300, 256, 256, 64), ("packed", 2100, 2100, 3, 1, 128)]                     # small blocks, pairs of tiles


def run(kernels, form, q, k, v, scale):
    """One sequence: q [new, H, hd], k and v [n, Hk, hd], causal."""
    kind, new, n, H, Hk, hd = form
    out = torch.full_like(q, 3.0)
    if kind == "packed":
        kernels.attention_packed(view(out), view(q), view(k), view(v), ints([0, n]), n, scale, MatmulMask.Causal)
    else:
        P = Pages(gen(n), [n], 32, Hk, hd)
        P.put(0, 0, k, v)
        kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints([0, new]), ints([n]), new, scale,
                                kernels.attention_paged_workspace(H, Hk, hd))
    kernels.device_status()
    return out


def first_column(n, H, hd, values):
    """[n, H, hd], zero but for the first column."""
    x = torch.zeros((n, H, hd), dtype=torch.float16, device="cuda")
    x[:, :, 0] = values.half()[:, None] if torch.is_tensor(values) else values
    return x


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("x", [9.5, 14.875, 17.0, 18.0])
def test_many_small_weights_count(kernels, form, x):
    """One key takes the most and all others e^-x of it each, as after a first token that every row looks at: together they
    are the output, because the first value is zero.

    Bound: a weight is rounded to fp16, 2^-11 of it, or 2^-32 of the row's largest where that is more; the exponential is
    good to 2^-18 and to 2^-21 of x; the sums' roundings, of 2^-24 each, are the factor 1.05; the output is rounded to
    fp16."""
    kind, new, n, H, Hk, hd = form
    big = 1024.0
    k = first_column(n, Hk, hd, torch.full((n,), -x, device="cuda"))
    k[0] = 0
    v = torch.full((n, Hk, hd), big, dtype=torch.float16, device="cuda")
    v[0] = 0
    out = run(kernels, form, first_column(new, H, hd, 1.0), k, v, 1.0)
    others = torch.arange(n - new, n, dtype=torch.float64, device="cuda")[:, None, None].expand(new, H, hd)
    p = math.exp(-x)
    l = 1 + others * p
    want = others * p * big / l
    tol = 1.05 * others * big / l * (max(p * 2.0 ** -11, 2.0 ** -32) + p * (2.0 ** -18 + 2.0 ** -21 * x)) \
        + want * 2.0 ** -11 + 2.0 ** -25
    assert_close(out, want, tol)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.088])
def test_scores_of_any_size(kernels, form, scale):
    """Scores of up to 10^11: whichever key is ahead takes the whole row, and nothing overflows.  (A product of 30000 and a
    multiple of 16 is exact in fp32; a sum of hd equal ones is off by hd * 2^-24 of it at most, 2 * 10^5 of 5.5 * 10^10 for
    head_dim 64 and four times as much for 128; two keys that differ do so by 16 * 30000 * hd, 3 and 6 * 10^7.)"""
    kind, new, n, H, Hk, hd = form
    g = gen(n + hd)
    step = torch.randperm(n, device="cuda", generator=g) % 3600 - 1800
    q = torch.full((new, H, hd), 30000.0, dtype=torch.float16, device="cuda")
    k = (step * 16).half()[:, None, None].expand(n, Hk, hd).contiguous()
    v = half(g, n, Hk, hd)
    out = run(kernels, form, q, k, v, scale)
    score = step.double() * (1 if scale > 0 else -1)
    for i in range(0, new, 1 + new // 40):
        seen = n - new + i + 1
        ahead = (score[:seen] == score[:seen].max()).nonzero().flatten()   # (equal keys share the row)
        want = v[ahead].double().mean(0).repeat_interleave(H // Hk, 0)
        size = v[ahead].double().abs().mean(0).repeat_interleave(H // Hk, 0)
        assert_close(out[i], want, size * 2.0 ** -11 * 1.05 + want.abs() * 2.0 ** -11 + 2.0 ** -25, i)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scale", [2.5e-3, 1.25e-3, 3e-4, -1e-5])
def test_scores_where_fp32_takes_steps_like_the_weights(kernels, form, scale):
    """Scores of 10^8 down to 10^6 with steps of 16 to 1/8 between them in fp32."""
    test_scores_of_any_size(kernels, form, scale)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("finite", [False, True])
def test_scores_of_minus_infinity(kernels, form, finite):
    """Keys with a score of -infinity have no weight; a row that sees no others has no softmax: not a number, in whichever
    kernel it is.  (Rows from the middle one on see keys of a finite score where there are such.)"""
    kind, new, n, H, Hk, hd = form
    k = first_column(n, Hk, hd, -INF)
    v = half(gen(n), n, Hk, hd)
    none = new // 2 if finite else new   # rows that see no finite score
    first = n - new + none
    k[first:] = 0
    out = run(kernels, form, first_column(new, H, hd, 1.0), k, v, 1.0)
    assert out[:none].isnan().all()
    rows = torch.arange(1, new - none + 1, device="cuda", dtype=torch.float64)[:, None, None]
    vs = v[first:].double()
    want = (vs.cumsum(0) / rows).repeat_interleave(H // Hk, 1)
    size = (vs.abs().cumsum(0) / rows).repeat_interleave(H // Hk, 1)
    # equal weights of 1, which fp16 holds; fp32 sums of up to 2100 of them
    assert_close(out[none:], want, size * 2100 * 2.0 ** -24 + size * 2.0 ** -11 + want.abs() * 2.0 ** -11 + 2.0 ** -25)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("value", [INF, -INF])
def test_infinite_scores_times_a_scale_of_zero(kernels, form, value):
    """0 * infinity is not a number: so are the rows that see that key, and no others."""
    kind, new, n, H, Hk, hd = form
    k = first_column(n, Hk, hd, 1.0)
    at = n - new + new // 2
    k[at, :, 0] = value
    v = half(gen(n), n, Hk, hd)
    out = run(kernels, form, first_column(new, H, hd, 1.0), k, v, 0.0)
    assert out[new // 2:].isnan().all() and out[:new // 2].isfinite().all()
