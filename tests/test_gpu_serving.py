"""The operators over sequences of different lengths against plain 64-bit forms (serving_oracle.py, which derives the
bounds), at the lengths, layouts and contents where they can go wrong."""
import math

import pytest
import torch

from adrastea_b200 import (AdrError, MatmulMask, RopeLayout, RopeScaling, TensorLayout, TensorView)
from serving_oracle import assert_close, attend, positions_of, rotate

pytestmark = pytest.mark.gpu
view = TensorView.of
NAN = float("nan")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).half()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ rotation
ROTATIONS = [  # tokens, heads, head_dim, rotary, half, scaling
    (1, 1, 2, 2, False, RopeScaling.Identity()),
    (3, 5, 128, 128, False, RopeScaling.Identity()),
    (7, 3, 64, 64, True, RopeScaling.Linear(4)),
    (5, 40, 128, 64, True, RopeScaling.Yarn(16, 8192)),
    (33, 2, 80, 80, True, RopeScaling.Base(2)),       # halves of 40 columns: whole pieces
    (9, 2, 96, 36, False, RopeScaling.Bands(8, 8192)),  # a part that ends inside a piece
    (9, 2, 96, 40, True, RopeScaling.Bands(8, 8192)),   # halves of 20 columns: no whole pieces
    (4, 3, 50, 10, True, RopeScaling.Identity()),
    (4, 3, 256, 254, False, RopeScaling.Identity()),
    (2, 64, 256, 256, True, RopeScaling.Yarn(4, 2048)),
]


@pytest.mark.parametrize("T,H,hd,rot,half_layout,scaling", ROTATIONS)
@pytest.mark.parametrize("pos0", [0, 126000, (1 << 31) - 40, -7])
def test_rope(kernels, T, H, hd, rot, half_layout, scaling, pos0):
    g = gen(T * hd + rot)
    x = half(g, T, H, hd)
    pos = (torch.arange(T, dtype=torch.int64) + pos0).to(torch.int32).cuda()
    table = kernels.rope_table(rot, 10000.0, RopeLayout.Half if half_layout else RopeLayout.Interleaved, scaling)
    out = torch.full_like(x, NAN)
    kernels.rope_f16(view(out), view(x), pos, table)
    want, tol = rotate(x, pos, rot, 10000.0, half_layout, scaling)
    assert_close(out, want, tol)
    assert torch.equal(out[..., rot:], x[..., rot:])
    # in place: the same bits
    kernels.rope_f16(view(x), view(x), pos, table)
    assert torch.equal(x, out)


@pytest.mark.parametrize("offset,pitch,head_first", [(0, 1000, False), (1, 333, False), (8, 336, False), (0, 0, True), (3, 0, True)])
@pytest.mark.parametrize("half_layout", [False, True])
def test_rope_of_strided_views(kernels, offset, pitch, head_first, half_layout):
    """Rows with a wider pitch, heads first, unaligned bases: only what the view covers is written."""
    T, H, hd = 11, 3, 64
    g = gen(offset + pitch)
    store = half(g, offset + T * max(pitch, H * hd) + 64)
    lay = TensorLayout.new((T, H, hd), (hd, T * hd, 1) if head_first else (pitch, hd, 1))
    src, before = TensorView(store, lay, offset), store.clone()
    pos = ints(list(range(100, 100 + T)))
    table = kernels.rope_table(64, 10000.0, RopeLayout(int(half_layout)))
    want, tol = rotate(src.as_torch().clone(), pos, 64, 10000.0, half_layout, RopeScaling())
    out = torch.full((T, H, hd), NAN, dtype=torch.float16, device="cuda")
    kernels.rope_f16(view(out), src, pos, table)
    assert torch.equal(store, before)
    assert_close(out, want, tol)
    kernels.rope_f16(src, src, pos, table)
    assert torch.equal(src.as_torch(), out)
    mask = torch.zeros_like(store, dtype=torch.bool)
    torch.as_strided(mask, lay.dims, lay.strides, offset).fill_(True)
    assert torch.equal(store[~mask], before[~mask])


def test_rope_agrees_with_the_plain_rotation(kernels):
    """Interleaved and unscaled it is the rotation of adr_rotary: both are within 2^-11 of the angle's formula, and near
    positions differ by one rounding at most."""
    g = gen(5)
    T, H, hd = 64, 8, 128
    x = half(g, T, H, hd)
    a, b = torch.empty_like(x), x.clone()
    kernels.rope_f16(view(a), view(x), ints(list(range(T))), kernels.rope_table(hd, 10000.0))
    kernels.rotary_inplace(view(b.view(T, H * hd)), H, 0, 10000.0)
    assert ((a - b).abs() <= 2.0 ** -10 * a.abs() + 2.0 ** -14).all()


# ------------------------------------------------------------------ pages
class Pages:
    """A pool of shuffled pages in one of three layouts, a table with junk behind the last page."""

    def __init__(self, g, lens, page, Hk, hd, layout="tokens", fill=NAN, extra=2):
        need = [-(-n // page) for n in lens]
        self.page, self.n = page, sum(need) + extra
        order = torch.randperm(self.n, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1) + 1), 1 << 30, dtype=torch.int32, device="cuda")
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m]
            at += m
        if layout == "tokens":
            self.k, self.v = (torch.full((self.n, page, Hk, hd), fill, dtype=torch.float16, device="cuda") for _ in "kv")
        elif layout == "heads":   # [page, head, slot, column]
            self.k, self.v = (torch.full((self.n, Hk, page, hd), fill, dtype=torch.float16, device="cuda").transpose(1, 2)
                              for _ in "kv")
        else:                     # k and v of a page next to each other
            both = torch.full((self.n, 2, page, Hk, hd), fill, dtype=torch.float16, device="cuda")
            self.k, self.v = both[:, 0], both[:, 1]

    def put(self, s, at, k, v):
        """k, v [m, Hk, hd] at positions at..at+m-1 of sequence s."""
        pos = torch.arange(at, at + k.shape[0], device="cuda")
        page = self.table[s].long()[pos // self.page]
        self.k[page, pos % self.page] = k
        self.v[page, pos % self.page] = v


APPENDS = [  # new, lens, H, Hk, hd, page, pool layout, rotary, half
    ([1], [1], 1, 1, 64, 16, "tokens", 64, False),
    ([1, 1, 1], [600, 17, 16], 32, 32, 128, 16, "tokens", 128, False),
    ([5, 0, 33, 1], [5, 40, 100, 33], 8, 2, 128, 32, "heads", 64, True),
    ([70, 2], [70, 300], 6, 3, 64, 64, "pairs", 24, True),
    ([3] * 40, list(range(3, 43)), 4, 1, 128, 16, "tokens", 128, True),
    ([2, 9], [7, 9], 3, 3, 40, 5, "tokens", 36, False),       # any page size, pairs one by one
    ([1] * 1100, [1 + i % 50 for i in range(1100)], 2, 1, 64, 16, "tokens", 64, False),
]


@pytest.mark.parametrize("new,lens,H,Hk,hd,page,layout,rot,half_layout", APPENDS)
def test_append(kernels, new, lens, H, Hk, hd, page, layout, rot, half_layout):
    g = gen(sum(lens) + hd)
    cu = starts(new)
    T = cu[-1] + 3  # three rows of no sequence
    qkv = half(g, T, H + 2 * Hk, hd)
    q, k, v = qkv.split([H, Hk, Hk], 1)
    P = Pages(g, lens, page, Hk, hd, layout, fill=7.0)
    q_out = torch.full((T, H, hd), NAN, dtype=torch.float16, device="cuda")
    scaling = RopeScaling.Yarn(4, 4096)
    table = kernels.rope_table(rot, 10000.0, RopeLayout(int(half_layout)), scaling)
    kernels.rope_append_paged(view(q_out), view(q), view(k), view(v), P.k, P.v, P.table, ints(cu), ints(lens), table)
    kernels.device_status()
    want_k, want_v = torch.full_like(P.k, 7.0), torch.full_like(P.v, 7.0)
    tol_k = torch.zeros(P.k.shape, dtype=torch.float64, device="cuda")
    exp_k = want_k.double()
    for s, (m, n) in enumerate(zip(new, lens)):
        if m == 0:
            continue
        rows = slice(cu[s], cu[s + 1])
        pos = torch.arange(n - m, n, device="cuda")
        wq, tq = rotate(q[rows], pos, rot, 10000.0, half_layout, scaling)
        assert_close(q_out[rows], wq, tq, "q")
        wk, tk = rotate(k[rows], pos, rot, 10000.0, half_layout, scaling)
        pg = P.table[s].long()[pos // page]
        exp_k[pg, pos % page], tol_k[pg, pos % page] = wk, tk
        want_v[pg, pos % page] = v[rows]
    assert_close(P.k, exp_k, tol_k, "k")
    assert torch.equal(P.v, want_v)
    assert q_out[cu[-1]:].isnan().all()
    # q in place: the same bits, k, v and the rows of no sequence kept
    before, q2 = qkv.clone(), q
    kernels.rope_append_paged(view(q2), view(q2), view(k), view(v), P.k, P.v, P.table, ints(cu), ints(lens), table)
    assert torch.equal(qkv[:cu[-1], :H], q_out[:cu[-1]]) and torch.equal(qkv[cu[-1]:], before[cu[-1]:])
    assert torch.equal(qkv[:, H:], before[:, H:])


def test_append_keeps_off_bad_pages(kernels):
    """Pages outside the pool, positions outside the table, before the first: nothing is written there, the status word
    says so, and the other rows are as ever."""
    g = gen(11)
    H, hd, page = 2, 64, 16
    new, lens = [2, 2, 3, 1], [20, 20, 2, 33]   # the third: a row at position -1; the fourth: past its two pages
    cu = starts(new)
    q, k, v = (half(g, cu[-1], H, hd) for _ in range(3))
    pool_k = torch.zeros((4, page, H, hd), dtype=torch.float16, device="cuda")
    pool_v = torch.zeros_like(pool_k)
    table = ints([[0, -1], [0, 4], [2, 1 << 30], [1, 1]])
    rope = kernels.rope_table(hd, 10000.0)
    out = torch.empty_like(q)
    kernels.rope_append_paged(view(out), view(q), view(k), view(v), pool_k, pool_v, table, ints(cu), ints(lens), rope)
    with pytest.raises(AdrError) as e:
        kernels.device_status()
    assert e.value.code == 5
    want = torch.zeros_like(pool_v)
    want[2, 0], want[2, 1] = v[5], v[6]
    assert torch.equal(pool_v, want) and not pool_k[[0, 1, 3]].any()
    pos = torch.tensor([18, 19, 18, 19, -1, 0, 1, 32], device="cuda")
    assert_close(out, *rotate(q, pos, hd, 10000.0, False, RopeScaling()))


# ------------------------------------------------------------------ packed prompts
PACKED = [  # lens, H, Hk, hd
    ([1], 1, 1, 64),
    ([1, 77, 3, 50], 4, 4, 64),
    ([5, 0, 0, 128, 129, 127], 2, 2, 128),
    ([257, 256, 255], 2, 1, 64),
    ([300, 1, 64], 10, 2, 128),     # five query heads to a key head
    ([600, 513], 3, 1, 128),
    ([16, 17, 15], 64, 1, 128),     # sixty-four to one
    ([2, 700], 14, 2, 64),
    ([1] * 70, 4, 2, 128),
    ([1300], 8, 1, 128),
    ([1024, 100], 4, 4, 128),
    ([30, 1, 77, 64] * 16, 16, 16, 64),   # more tiles than two CTAs to an SM: blocks of 64 keys
    ([257] * 7, 16, 16, 64),
    ([200, 129, 65], 128, 128, 64),
    ([2100, 50], 2, 1, 64),
    ([2100, 50], 4, 1, 128),              # two tiles to a CTA
    ([300] * 40, 2, 2, 64),               # more sequences than a warp has lanes
    ([129, 130, 131, 132, 133, 257], 2, 1, 64),             # a few keys behind a full block
    ([65, 130, 195, 260, 69, 129, 2, 64] * 8, 16, 16, 64),
]


def check_packed(kernels, lens, H, Hk, hd, causal, q, k, v, out, cu=None, scale=None):
    cu = cu or starts(lens)
    scale = scale or 1.0 / math.sqrt(hd)
    kernels.attention_packed(view(out), view(q), view(k), view(v), ints(cu), max(max(lens), 1), scale,
                             MatmulMask.Causal if causal else MatmulMask.None_)
    kernels.device_status()
    for s, n in enumerate(lens):
        rows = slice(cu[s], cu[s + 1])
        want, tol = attend(q[rows], k[rows], v[rows], scale, 1 if causal else None)
        assert_close(out[rows], want, tol, (s, n))


@pytest.mark.parametrize("lens,H,Hk,hd", PACKED)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("fused", [True, False])
def test_packed(kernels, lens, H, Hk, hd, causal, fused):
    g = gen(sum(lens) * 3 + H)
    T = sum(lens) + 5  # rows of no sequence, in q and k and v not a number
    if fused:
        q, k, v = half(g, T, H + 2 * Hk, hd).split([H, Hk, Hk], 1)
    else:
        q, k, v = half(g, T, H, hd), half(g, Hk, T, hd).transpose(0, 1), half(g, T, Hk, hd)
    for t in (q, k, v):
        t[sum(lens):] = NAN
    out = torch.full((T, H, hd), 3.0, dtype=torch.float16, device="cuda")
    check_packed(kernels, lens, H, Hk, hd, causal, q, k, v, out)
    assert (out[sum(lens):] == 3.0).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_sequences_do_not_touch_each_other(kernels, hd, causal):
    """Infinities and NaN in one sequence stay in it; rows before the first sequence are left alone."""
    g = gen(hd)
    lens, H, Hk = [40, 130, 33, 200], 4, 2
    cu = starts(lens)
    q, k, v = half(g, cu[-1], H, hd), half(g, cu[-1], Hk, hd), half(g, cu[-1], Hk, hd)
    for s in (0, 2):
        k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]] = NAN, float("inf")
    out = torch.full_like(q, 5.0)
    kernels.attention_packed(view(out), view(q), view(k), view(v), ints([40] + cu[2:]), 200, 0.1,
                             MatmulMask.Causal if causal else MatmulMask.None_)
    kernels.device_status()
    assert (out[:40] == 5.0).all() and out[cu[2]:cu[3]].isnan().all()
    for s in (1, 3):
        rows = slice(cu[s], cu[s + 1])
        assert_close(out[rows], *attend(q[rows], k[rows], v[rows], 0.1, 1 if causal else None))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,n", [(2, 2, 300), (8, 1, 300), (256, 256, 300), (3, 1, 2100)])  # every form of tile
@pytest.mark.parametrize("at", [0, 20, 150, 299])
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_packed_rows_before_a_bad_token_do_not_see_it(kernels, hd, H, Hk, n, at, value):
    """k and v of one token are not finite: causal rows before it are as if they were, rows from it on see it."""
    g = gen(at + hd)
    q, k, v = half(g, n, H, hd), half(g, n, Hk, hd), half(g, n, Hk, hd)
    clean_k, clean_v = k.clone(), v.clone()
    v[at, :, 3] = value
    out = torch.empty_like(q)
    kernels.attention_packed(view(out), view(q), view(k), view(v), ints([0, n]), n, 0.1)
    want, tol = attend(q, clean_k, clean_v, 0.1, 1)
    other = [c for c in range(hd) if c != 3]
    assert_close(out[:at], want[:at], tol[:at], "before")
    assert_close(out[..., other], want[..., other], tol[..., other], "other columns")
    if math.isnan(value):
        assert out[at:, :, 3].isnan().all()
    else:  # its weight times infinity; 0 * infinity where the 16-bit weight vanishes
        assert not out[at:, :, 3].isfinite().any()
    k[at] = value
    kernels.attention_packed(view(out), view(q), view(k), view(v), ints([0, n]), n, 0.1)
    assert_close(out[:at], want[:at], tol[:at], "key")
    assert out[at].isnan().all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", [2, 256])
def test_packed_large_scores(kernels, H, hd):
    """Maxima that grow along the keys by hundreds, falling ones, and equal ones; a negative scale and zero."""
    n = 520
    g = gen(1)
    for kind in ("grow", "fall", "equal", "negative", "zero"):
        q, k, v = half(g, n, H, hd), half(g, n, H, hd), half(g, n, H, hd)
        ramp = torch.linspace(-4, 4, n, device="cuda")[:, None, None]
        if kind in ("grow", "fall"):
            q = torch.ones_like(q)
            k = ((ramp if kind == "grow" else -ramp) + 0.1 * k.float()).half()
        if kind == "equal":
            k = k[:1].expand(n, H, hd).contiguous()
        scale = {"negative": -0.2, "zero": 0.0}.get(kind, 0.7)
        out = torch.empty_like(q)
        kernels.attention_packed(view(out), view(q), view(k), view(v), ints([0, n]), n, scale)
        assert_close(out, *attend(q, k, v, scale, 1), kind)


@pytest.mark.parametrize("n,S", [(258, 1), (260, 20)])
def test_packed_last_keys_of_every_size(kernels, n, S):
    """The keys behind the last full block have the largest scores, the smallest, or equal ones; a negative scale, zero; one of
    them, or its value, is not finite, which every row sees."""
    H, hd = 16, 64
    g = gen(n)
    for kind in ("largest", "smallest", "equal", "negative", "zero", "key", "value"):
        q, k, v = (half(g, S, n, H, hd) for _ in "qkv")
        if kind in ("largest", "smallest"):
            q = torch.ones_like(q)
            k[:, 256:] = 5.0 if kind == "largest" else -5.0
        if kind == "equal":
            k = k[:, :1].expand(S, n, H, hd).contiguous()
        if kind == "key":
            k[:, n - 1, 0] = NAN
        if kind == "value":
            v[:, n - 1, 0, 3] = float("inf")
        scale = {"negative": -0.2, "zero": 0.0}.get(kind, 0.3)
        out = torch.empty_like(q)
        kernels.attention_packed(view(out.view(S * n, H, hd)), view(q.view(S * n, H, hd)), view(k.view(S * n, H, hd)),
                                 view(v.view(S * n, H, hd)), ints([n * s for s in range(S + 1)]), n, scale, MatmulMask.None_)
        if kind == "key":
            assert out[:, :, 0].isnan().all()
            out, q, k, v = (t[:, :, 1:] for t in (out, q, k, v))
        if kind == "value":
            assert (out[:, :, 0, 3] == float("inf")).all()
            v[:, n - 1, 0, 3] = out[:, :, 0, 3] = 0.0
        for s in range(0, S, 5):
            want, tol = attend(q[s], k[s], v[s], scale, None)
            if kind == "value":
                want[:, 0, 3] = 0.0
            assert_close(out[s], want, tol, (kind, s))


def test_packed_wrong_spans_stay_inside(kernels):
    """cu_q outside the rows: the spans are cut to the rows there are, and nothing outside is touched; where it falls,
    the sequence has no rows."""
    g = gen(2)
    T, H, hd = 100, 2, 64
    store = half(g, 3, T + 20, H, hd)
    q, k, v = store[:, 10:-10]
    out = torch.full((T + 20, H, hd), 2.0, dtype=torch.float16, device="cuda")
    kernels.attention_packed(view(out[10:-10]), view(q), view(k), view(v), ints([-50, 30, 20, 30, 1000]), 100, 0.1)
    kernels.device_status()
    assert (out[:10] == 2.0).all() and (out[-10:] == 2.0).all()
    assert_close(out[10:30], *[t[:20] for t in attend(q[:30], k[:30], v[:30], 0.1, 1)])
    assert_close(out[40:-10], *attend(q[30:], k[30:], v[30:], 0.1, 1))


# ------------------------------------------------------------------ paged attention
PAGED = [  # new, lens, H, Hk, hd, page, pool layout
    ([1], [1], 1, 1, 64, 16, "tokens"),
    ([1], [600], 32, 32, 128, 16, "tokens"),
    ([1, 1, 1, 1], [1, 64, 65, 1000], 8, 2, 128, 16, "tokens"),
    ([1, 1], [5000, 3], 64, 8, 128, 64, "heads"),
    ([1] * 9, [17 * i + 1 for i in range(9)], 14, 2, 64, 32, "pairs"),
    ([4, 1, 0, 3], [100, 1, 50, 700], 20, 4, 128, 128, "tokens"),
    ([8, 8], [8, 1025], 8, 1, 64, 256, "tokens"),
    ([9, 2, 17], [400, 2, 17], 32, 8, 128, 16, "heads"),
    ([130, 1, 40], [1200, 900, 40], 8, 2, 128, 16, "tokens"),
    ([300], [300], 4, 4, 64, 64, "pairs"),
    ([257, 64], [2000, 65], 10, 2, 128, 256, "tokens"),
    ([1, 500, 1, 33], [3000, 800, 70, 33], 16, 2, 64, 32, "tokens"),
    ([1] * 200, [1 + (i * 37) % 300 for i in range(200)], 4, 1, 64, 16, "tokens"),
    ([2], [9000], 64, 1, 128, 128, "tokens"),
    ([64], [20000], 8, 8, 64, 64, "tokens"),
    ([100, 7], [6000, 6000], 2, 1, 128, 16, "heads"),
    ([40, 300, 33, 100, 41, 64, 50, 90], [900, 300, 33, 2000, 41, 640, 129, 1000], 16, 16, 128, 16, "tokens"),  # pairs of tiles
    ([100, 40, 77] * 4, [400, 40, 128] * 4, 16, 16, 128, 32, "pairs"),       # single tiles
    ([40, 300, 33, 100, 41, 64, 50, 90], [900, 300, 33, 2000, 41, 640, 129, 1000], 16, 16, 64, 64, "heads"),
    ([3, 8], [3, 2000], 64, 16, 64, 16, "tokens"),                            # 32 rows of a key head
    ([33], [30000], 1, 1, 128, 256, "tokens"),                                # keys shared out among CTAs
    ([50, 1, 1, 60], [9000, 9000, 1, 60], 8, 2, 64, 128, "pairs"),
    ([1, 300, 1, 33, 200] * 3, [500, 300, 90, 700, 201] * 3, 32, 32, 64, 32, "tokens"),   # both kernels, whole tiles
    ([1, 100, 100], [9000, 300, 100], 32, 32, 128, 64, "tokens"),                         # both, keys shared out
]


def paged_case(new, lens, H, Hk, hd, page, layout, seed=0, spare=3):
    g = gen(sum(lens) + hd + seed)
    cu = starts(new)
    q = half(g, cu[-1] + spare, H, hd)
    P = Pages(g, lens, page, Hk, hd, layout)  # slots that nothing was put into are not a number
    kv = [(half(g, n, Hk, hd), half(g, n, Hk, hd)) for n in lens]
    for s, (k, v) in enumerate(kv):
        P.put(s, 0, k, v)
    return q, P, kv, cu


@pytest.mark.parametrize("new,lens,H,Hk,hd,page,layout", PAGED)
@pytest.mark.parametrize("hint", ["longest", "one", "many"])
def test_paged(kernels, new, lens, H, Hk, hd, page, layout, hint):
    """`hint`: max_q as it is, or wrong: it may cost time, not the result."""
    q, P, kv, cu = paged_case(new, lens, H, Hk, hd, page, layout)
    scale = 1.0 / math.sqrt(hd)
    out = torch.full_like(q, 3.0)
    ws = kernels.attention_paged_workspace(H, Hk, hd)
    max_q = {"longest": max(new), "one": 1, "many": 4096}[hint]
    ws.fill_(255)
    for _ in range(2):  # the second call finds the first one's workspace
        out.fill_(3.0)
        kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints(lens), max_q, scale, ws)
    kernels.device_status()
    for s, (m, n) in enumerate(zip(new, lens)):
        rows = slice(cu[s], cu[s + 1])
        want, tol = attend(q[rows], *kv[s], scale, n - m + 1)
        assert_close(out[rows], want, tol, (s, m, n))
    assert (out[cu[-1]:] == 3.0).all()


@pytest.mark.parametrize("new,lens", [([5], [2]), ([3, 1], [0, 0]), ([40, 1], [10, 30]), ([200], [100])])
@pytest.mark.parametrize("hd", [64, 128])
def test_paged_rows_that_see_nothing_are_zeros(kernels, new, lens, hd):
    """More rows than positions: the first rows lie before position 0.  No positions at all: all of them."""
    H, Hk = 4, 2
    q, P, kv, cu = paged_case(new, lens, H, Hk, hd, 16, "tokens")
    out = torch.full_like(q, NAN)
    kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints(lens), max(new), 0.2,
                            kernels.attention_paged_workspace(H, Hk, hd))
    for s, (m, n) in enumerate(zip(new, lens)):
        rows = slice(cu[s], cu[s + 1])
        want, tol = attend(q[rows], *kv[s], 0.2, n - m + 1)
        assert_close(out[rows], want, tol)
        assert not out[cu[s]:cu[s] + max(0, m - n)].any()


@pytest.mark.parametrize("new,n,H,Hk", [(6, 400, 8, 2), (20, 300, 1, 1), (150, 400, 8, 2), (150, 3000, 8, 2), (600, 700, 32, 16)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [NAN, float("inf"), float("-inf")])
def test_paged_rows_before_a_bad_token_do_not_see_it(kernels, new, n, H, Hk, hd, value):
    for at in (n - new + 2, n - 1):
        q, P, kv, cu = paged_case([new], [n], H, Hk, hd, 32, "tokens", seed=at)
        k, v = kv[0]
        want, tol = attend(q[:new], k, v, 0.1, n - new + 1)
        v[at, :, 5] = value
        P.put(0, 0, k, v)
        out, ws = torch.empty_like(q), kernels.attention_paged_workspace(H, Hk, hd)
        kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints([n]), new, 0.1, ws)
        first = at - (n - new)
        assert_close(out[:first], want[:first], tol[:first])
        other = [c for c in range(hd) if c != 5]
        assert_close(out[:new, :, other], want[..., other], tol[..., other])
        assert not out[first:new, :, 5].isfinite().any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,n,H,Hk", [(1, 900, 8, 2), (7, 900, 4, 1), (90, 900, 4, 1), (90, 5000, 4, 1)])  # every kernel
def test_paged_large_scores(kernels, new, n, H, Hk, hd):
    """Maxima that grow and fall along the keys by hundreds, equal ones; a negative scale and zero."""
    for kind in ("grow", "fall", "equal", "negative", "zero"):
        q, P, kv, cu = paged_case([new], [n], H, Hk, hd, 32, "tokens", seed=7)
        k, v = kv[0]
        ramp = torch.linspace(-4, 4, n, device="cuda")[:, None, None]
        if kind in ("grow", "fall"):
            q = torch.ones_like(q)
            k = ((ramp if kind == "grow" else -ramp) + 0.1 * k.float()).half()
        if kind == "equal":
            k = k[:1].expand(n, Hk, hd).contiguous()
        P.put(0, 0, k, v)
        scale = {"negative": -0.2, "zero": 0.0}.get(kind, 0.7)
        out, ws = torch.empty_like(q), kernels.attention_paged_workspace(H, Hk, hd)
        kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints([n]), new, scale, ws)
        assert_close(out[:new], *attend(q[:new], k, v, scale, n - new + 1), kind)


@pytest.mark.parametrize("new", [1, 3])
def test_many_sequences(kernels, new):
    """More sequences than a warp looks up at once, twice over: appended, attended over pages, and packed."""
    S, H, Hk, hd, page = 1500, 2, 1, 64, 16
    lens = [new + (i * 7) % 40 for i in range(S)]
    q, P, kv, cu = paged_case([new] * S, lens, H, Hk, hd, page, "tokens")
    rope = kernels.rope_table(hd, 10000.0)
    pos = torch.tensor([n - new + i for n in lens for i in range(new)], device="cuda")
    g = gen(3)
    k, v = half(g, cu[-1], Hk, hd), half(g, cu[-1], Hk, hd)
    turned_q, turned_k, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    at = pos.int()
    kernels.rope_f16(view(turned_q[:cu[-1]]), view(q[:cu[-1]]), at, rope)
    kernels.rope_f16(view(turned_k), view(k), at, rope)
    rows = torch.empty_like(q)
    kernels.rope_append_paged(view(rows[:cu[-1]]), view(q[:cu[-1]]), view(k), view(v), P.k, P.v, P.table, ints(cu), ints(lens),
                              rope)
    assert torch.equal(rows[:cu[-1]], turned_q[:cu[-1]])
    ws = kernels.attention_paged_workspace(H, Hk, hd)
    kernels.attention_paged(view(out), view(rows), P.k, P.v, P.table, ints(cu), ints(lens), new, 0.1, ws)
    packed = torch.empty_like(rows[:cu[-1]])
    kernels.attention_packed(view(packed), view(rows[:cu[-1]]), view(turned_k), view(v), ints(cu), new, 0.1)
    kernels.device_status()
    for s in range(0, S, 7):
        mine = slice(cu[s], cu[s + 1])
        keys, values = (torch.cat([old[:lens[s] - new], fresh[mine]]) for old, fresh in zip(kv[s], (turned_k, v)))
        assert_close(out[mine], *attend(rows[mine], keys, values, 0.1, lens[s] - new + 1), s)
        assert_close(packed[mine], *attend(rows[mine], turned_k[mine], v[mine], 0.1, 1), s)


@pytest.mark.parametrize("n,T,positions", [(64, 64, 128), (1025, 2048, 262144)])
def test_paged_overlapping_sequences_are_left_undone(kernels, n, T, positions):
    """Every second sequence claims all rows: more work than sequences side by side can have (of the larger case, more
    than 32 bits count).  Nothing is written and the status word says so; the workspace is fit for the next call."""
    H, Hk, hd, page = 32, 8, 64, 16
    q = half(gen(n), T, H, hd)
    pool = torch.zeros((1, page, Hk, hd), dtype=torch.float16, device="cuda")
    table = torch.zeros((n, positions // page), dtype=torch.int32, device="cuda")
    out, ws = torch.full_like(q, 2.0), kernels.attention_paged_workspace(H, Hk, hd)
    cu, lens = ints([T * (s % 2) for s in range(n + 1)]), ints([positions] * n)
    kernels.attention_paged(view(out), view(q), pool, pool, table, cu, lens, 8, 0.1, ws)
    with pytest.raises(AdrError) as e:
        kernels.device_status()
    assert e.value.code == 5 and (out == 2.0).all()
    q, P, kv, cu = paged_case([3], [50], H, Hk, hd, page, "tokens", seed=1)
    out = torch.empty_like(q)
    kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints([50]), 3, 0.1, ws)
    assert_close(out[:3], *attend(q[:3], *kv[0], 0.1, 48))


@pytest.mark.parametrize("new", [1, 90])
def test_paged_bad_pages_read_as_zeros(kernels, new):
    """A page outside the pool, a length past the table: zeros and a status, no access."""
    n, H, Hk, hd, page = 200, 4, 2, 128, 16
    q, P, kv, cu = paged_case([new], [n], H, Hk, hd, page, "tokens")
    for wrong in (-1, P.n, (1 << 31) - 1, -(1 << 31)):
        table = P.table.clone()
        table[0, 3] = wrong
        k, v = (torch.nan_to_num(positions_of(t, table[0], n)) for t in (P.k, P.v))
        out, ws = torch.full_like(q, NAN), kernels.attention_paged_workspace(H, Hk, hd)
        kernels.attention_paged(view(out), view(q), P.k, P.v, table, ints(cu), ints([n]), new, 0.1, ws)
        with pytest.raises(AdrError) as e:
            kernels.device_status()
        assert e.value.code == 5
        assert_close(out[:new], *attend(q[:new], k, v, 0.1, n - new + 1))
    table = P.table[:, :5].contiguous()  # 80 positions of 200
    out = torch.full_like(q, NAN)
    kernels.attention_paged(view(out), view(q), P.k, P.v, table, ints(cu), ints([n]), new, 0.1, ws)
    with pytest.raises(AdrError):
        kernels.device_status()
    k, v = (t[:80] for t in kv[0])
    assert_close(out[:new], *attend(q[:new], k, v, 0.1, 80 - new + 1))


@pytest.mark.parametrize("new", [1, 130])
def test_paged_offsets_past_32_bits(kernels, new):
    """A pool of more than 2^31 elements, the sequence at its far end; k and v are the same pool."""
    hd, Hk, H, page = 128, 8, 16, 256
    n_pages = (1 << 31) // (hd * Hk * page) + 40
    pool = torch.zeros((n_pages, page, Hk, hd), dtype=torch.float16, device="cuda")
    g = gen(4)
    n = 1500
    need = -(-n // page)
    idx = torch.randperm(20, device="cuda", generator=g)[:need] + n_pages - 20
    k = half(g, n, Hk, hd)
    q, rope = half(g, new, H, hd), kernels.rope_table(hd, 10000.0)
    table = idx.to(torch.int32)[None].contiguous()
    pos = torch.arange(n, device="cuda")
    pool[idx[pos // page], pos % page] = k
    out = torch.empty_like(q)
    ws = kernels.attention_paged_workspace(H, Hk, hd)
    kernels.attention_paged(view(out), view(q), pool, pool, table, ints([0, new]), ints([n]), new, 0.1, ws)
    kernels.device_status()
    assert_close(out, *attend(q, k, k, 0.1, n - new + 1))
    kk, vv = half(g, new, Hk, hd), half(g, new, Hk, hd)
    kernels.rope_append_paged(view(out), view(q), view(kk), view(vv), pool, pool, table, ints([0, new]), ints([n]), rope)
    at = torch.arange(n - new, n, device="cuda")
    got = pool[idx[at // page], at % page]
    # k and v went to the same slots: every element is one or the other's
    wk, tk = rotate(kk, at, hd, 10000.0, False, RopeScaling())
    assert (((got.double() - wk).abs() <= tk) | (got == vv)).all()


# ------------------------------------------------------------------ run together
def chain(kernels, st):
    """One serving step: rotation and append, then attention over the cache."""
    H, Hk = st["H"], st["Hk"]
    q, k, v = st["qkv"].split([H, Hk, Hk], 1)
    kernels.rope_append_paged(view(st["q"]), view(q), view(k), view(v), st["P"].k, st["P"].v, st["P"].table, st["cu"],
                              st["lens"], st["rope"])
    kernels.attention_paged(view(st["out"]), view(st["q"]), st["P"].k, st["P"].v, st["P"].table, st["cu"], st["lens"],
                            st["max_q"], st["scale"], st["ws"])


@pytest.mark.parametrize("pdl", [0, 1])
@pytest.mark.parametrize("hd,H,Hk", [(64, 4, 4), (128, 8, 2)])
def test_prompt_chunks_and_tokens_are_one_attention(kernels, pdl, hd, H, Hk):
    """A sequence that goes through the cache as a prompt, a chunk and single tokens, beside another that starts later,
    gets what attention_packed over the whole rotated sequence gives (both are within their bounds of the formula)."""
    kernels.set_tunable("pdl", pdl)
    try:
        g = gen(hd + pdl)
        total = [211, 150]
        qkv = [half(g, n, H + 2 * Hk, hd) for n in total]
        rope = kernels.rope_table(hd, 10000.0, RopeLayout.Half)
        P = Pages(g, total, 16, Hk, hd)
        steps = [(130, 0), (70, 64)] + [(1, 1)] * 11 + [(0, 75)]
        at = [0, 0]
        got = [[], []]
        ws = kernels.attention_paged_workspace(H, Hk, hd)
        for new in steps:
            rows = torch.cat([qkv[s][at[s]:at[s] + new[s]] for s in (0, 1)])
            at = [a + n for a, n in zip(at, new)]
            T = sum(new)
            st = dict(H=H, Hk=Hk, qkv=rows, q=torch.empty((T, H, hd), dtype=torch.float16, device="cuda"), P=P,
                      cu=ints(starts(new)), lens=ints(at), rope=rope, max_q=max(new), scale=0.11, ws=ws,
                      out=torch.empty((T, H, hd), dtype=torch.float16, device="cuda"))
            chain(kernels, st)
            for s, part in enumerate(st["out"].split(list(new))):
                got[s].append(part)
        cu = starts(total)
        rows = torch.cat(qkv)
        q, k, v = rows.split([H, Hk, Hk], 1)
        pos = torch.cat([torch.arange(n, device="cuda") for n in total]).to(torch.int32)
        kernels.rope_f16(view(rows[:, :H + Hk]), view(rows[:, :H + Hk]), pos, rope)
        out = torch.empty((cu[-1], H, hd), dtype=torch.float16, device="cuda")
        kernels.attention_packed(view(out), view(q), view(k), view(v), ints(cu), max(total), 0.11)
        kernels.device_status()
        for s in (0, 1):
            part = slice(cu[s], cu[s + 1])
            want, tol = attend(q[part], k[part], v[part], 0.11, 1)
            assert_close(torch.cat(got[s]), want, tol, "paged")
            assert_close(out[part], want, tol, "packed")
    finally:
        kernels.set_tunable("pdl", 0)


@pytest.mark.parametrize("pdl", [0, 1])
def test_a_captured_step_is_replayed_with_other_lengths(kernels, pdl):
    """Lengths, tables, q, k and v change between replays; two graphs use one workspace, one after the other."""
    kernels.set_tunable("pdl", pdl)
    try:
        H, Hk, hd, page, n = 8, 2, 128, 16, 3
        g = gen(9)
        P = Pages(g, [2000] * n, page, Hk, hd, fill=0.0)
        P.k.copy_(half(g, *P.k.shape))
        P.v.copy_(half(g, *P.v.shape))
        ws = kernels.attention_paged_workspace(H, Hk, hd)
        graphs = []
        for T, max_q in ((n, 1), (2 * n, 2)):
            st = dict(H=H, Hk=Hk, qkv=half(g, T, H + 2 * Hk, hd), q=torch.empty((T, H, hd), dtype=torch.float16, device="cuda"),
                      P=P, cu=ints([i * T // n for i in range(n + 1)]), lens=ints([100] * n),
                      rope=kernels.rope_table(hd, 10000.0), max_q=max_q, scale=0.1, ws=ws,
                      out=torch.empty((T, H, hd), dtype=torch.float16, device="cuda"))
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                chain(kernels, st)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                chain(kernels, st)
            graphs.append((graph, st, T // n))
        for lens in ([100, 100, 100], [2, 1999, 64], [2000, 1000, 1], [5, 6, 7]):
            lens = [max(x, 2) for x in lens]
            for graph, st, m in graphs:
                st["lens"].copy_(ints(lens))
                st["qkv"].copy_(half(g, *st["qkv"].shape))
                graph.replay()
                torch.cuda.synchronize()
                for s in range(n):
                    k, v = (positions_of(t, P.table[s], lens[s]) for t in (P.k, P.v))
                    rows = slice(s * m, (s + 1) * m)
                    assert_close(st["out"][rows], *attend(st["q"][rows], k, v, 0.1, lens[s] - m + 1))
        kernels.device_status()
    finally:
        kernels.set_tunable("pdl", 0)


def test_calls_on_two_streams_at_once(kernels):
    """A workspace each: both are right, and on a stream that is not the current one."""
    g = gen(21)
    jobs = []
    for i, (H, Hk, hd) in enumerate([(32, 8, 128), (16, 16, 64)]):
        new, lens = [1] * 6, [3000, 10, 500, 1500, 64, 2000]
        q, P, kv, cu = paged_case(new, lens, H, Hk, hd, 32, "tokens", seed=i)
        jobs.append((torch.cuda.Stream(), q, P, kv, cu, lens, torch.empty_like(q), kernels.attention_paged_workspace(H, Hk, hd)))
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, q, P, kv, cu, lens, out, ws in jobs:
            kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), ints(lens), 1, 0.1, ws, stream=stream)
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    kernels.device_status()
    for stream, q, P, kv, cu, lens, out, ws in jobs:
        for s, n in enumerate(lens):
            assert_close(out[s:s + 1], *attend(q[s:s + 1], *kv[s], 0.1, n))


def test_results_do_not_change_from_call_to_call(kernels):
    q, P, kv, cu = paged_case([1] * 5, [9000, 20, 4000, 777, 6001], 32, 8, 128, 16, "tokens")
    lens, ws = ints([9000, 20, 4000, 777, 6001]), kernels.attention_paged_workspace(32, 8, 128)
    outs = []
    for _ in range(4):
        out = torch.empty_like(q)
        kernels.attention_paged(view(out), view(q), P.k, P.v, P.table, ints(cu), lens, 1, 0.1, ws)
        outs.append(out[:5])
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_python_side_refuses(kernels):
    """Wrong types, devices and shapes are refused before a launch."""
    H, Hk, hd = 4, 2, 64
    q, k = torch.zeros((6, H, hd), dtype=torch.float16, device="cuda"), torch.zeros((6, Hk, hd), dtype=torch.float16, device="cuda")
    pool = torch.zeros((4, 16, Hk, hd), dtype=torch.float16, device="cuda")
    cu, lens, table = ints([0, 2, 6]), ints([10, 20]), ints([[0, 1], [2, 3]])
    ws, rope = kernels.attention_paged_workspace(H, Hk, hd), kernels.rope_table(hd, 10000.0)
    n = kernels.launch_count()
    paged = lambda **c: kernels.attention_paged(*[c.get(a, b) for a, b in dict(
        out=view(q), q=view(q), k=pool, v=pool, table=table, cu=cu, lens=lens, max_q=4, scale=0.1, ws=ws).items()])
    for change, error in [(dict(out=view(q.float())), TypeError), (dict(q=view(q.cpu())), AssertionError),
                          (dict(k=pool.bfloat16()), TypeError), (dict(v=pool[:, :, :1]), AssertionError),
                          (dict(table=table.long()), TypeError), (dict(table=table[:, :1]), AssertionError),
                          (dict(cu=cu[:2]), AssertionError), (dict(lens=lens.cpu()), AssertionError),
                          (dict(ws=ws[:-1]), AdrError), (dict(max_q=0), AdrError), (dict(table=ints([[0, 1]])), AssertionError),
                          (dict(out=view(q[:, :2])), AssertionError)]:
        with pytest.raises(error):
            paged(**change)
    with pytest.raises(AssertionError):
        kernels.rope_f16(view(q), view(q), ints([1, 2]), rope)
    with pytest.raises(TypeError):
        kernels.rope_f16(view(q), view(q), ints([1] * 6).long(), rope)
    with pytest.raises(AssertionError):
        kernels.attention_packed(view(q), view(q), view(k), view(k[:, :1]), cu, 4, 0.1)
    with pytest.raises(AdrError):
        kernels.attention_packed(view(q), view(q), view(k), view(k), cu, 4, float("nan"))
    assert kernels.launch_count() == n
