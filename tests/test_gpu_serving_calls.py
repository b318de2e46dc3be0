"""Calls of the serving operators that the documentation allows: the captured and the concurrent ones with every output
checked against what went in, the largest sizes, arrays that contradict one another."""
import pytest
import torch

from adrastea_b200 import AdrError, RopeLayout, RopeScaling
from adrastea_b200.llama import LlamaShape, LlamaU8
from serving_oracle import assert_close, attend, positions_of, rotate
from test_gpu_serving import Pages, chain, gen, half, ints, paged_case, starts, view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("n,T,H,Hk,hd", [(64, 2048, 32, 8, 64), (31, 2048, 8, 8, 128), (200, 300, 4, 4, 64), (9, 130, 2, 1, 128)])
def test_tiles_of_overlapping_sequences(kernels, paged, n, T, H, Hk, hd):
    """Every second sequence claims all rows: more tiles than sequences side by side can have.  What is written are rows of
    those sequences, nothing beside them; the next call is as ever."""
    g, page = gen(n), 16
    q, k, v = half(g, T, H, hd), half(g, T, Hk, hd), half(g, T, Hk, hd)
    P = Pages(g, [1024], page, Hk, hd)
    keys, values = half(g, 1024, Hk, hd), half(g, 1024, Hk, hd)
    P.put(0, 0, keys, values)
    table = P.table[:, :-1].expand(n, -1).contiguous()
    store, ws = torch.full((T + 20, H, hd), 2.0, dtype=torch.float16, device="cuda"), kernels.attention_paged_workspace(H, Hk, hd)
    out = store[10:-10]

    def call(cu, lens, max_q):
        if paged:
            kernels.attention_paged(view(out), view(q), P.k, P.v, table, ints(cu), ints(lens), max_q, 0.1, ws)
        else:
            kernels.attention_packed(view(out), view(q), view(k), view(v), ints(cu), max_q, 0.1)

    def check(rows, may_be_undone):
        m = rows.stop - rows.start
        want, tol = attend(q[rows], *((keys, values, 0.1, 1024 - m + 1) if paged else (k[rows], v[rows], 0.1, 1)))
        done = (out[rows] != 2.0).any(-1, keepdim=True) if may_be_undone else torch.ones_like(want[..., :1], dtype=torch.bool)
        assert_close(torch.where(done, out[rows].double(), 0.0), torch.where(done, want, 0.0), tol)

    call([T * (s % 2) for s in range(n + 1)], [1024] * n, T)
    try:
        kernels.device_status()   # (it may say so, and need not)
    except AdrError:
        pass
    check(slice(0, T), True)
    cu = [T * s // n for s in range(n + 1)]
    call(cu, [1024] * n, max(b - a for a, b in zip(cu, cu[1:])))
    kernels.device_status()
    for a, b in zip(cu, cu[1:]):
        check(slice(a, b), False)
    assert (store[:10] == 2.0).all() and (store[-10:] == 2.0).all()


def test_as_many_rows_as_there_are_positions(kernels):
    """2^31 - 1 rows in one call (34 GB, in place)."""
    T = (1 << 31) - 1
    g = gen(8)
    x = torch.zeros((T, 1, 8), dtype=torch.float16, device="cuda")
    ends = [slice(0, 5), slice(T - 5, T)]
    before = [half(g, 5, 1, 8) for _ in ends]
    for at, b in zip(ends, before):
        x[at] = b
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    table = kernels.rope_table(8, 10000.0, RopeLayout.Interleaved)
    kernels.rope_f16(view(x), view(x), pos, table)
    for at, b in zip(ends, before):
        assert_close(x[at], *rotate(b, pos[at], 8, 10000.0, False, RopeScaling()))
    del x, pos
    torch.cuda.empty_cache()


@pytest.mark.parametrize("captured", [False, True])
def test_logits_of_a_step_do_not_see_those_of_the_step_before(kernels, captured):
    """A request whose logits are not numbers does not spoil the next one in its row of the output: not of `extend`, not of
    a new prompt, not of a token of the rectangular cache."""
    shape = LlamaShape(dim=256, n_heads=2, ffn=512, n_layers=1, vocab=512, block=64)
    toks = torch.randint(0, shape.vocab, (2, 9), device="cuda", generator=gen(1))
    bad = torch.full((2, 1), 3, dtype=torch.int64, device="cuda")

    def run(spoil):
        model = LlamaU8(kernels, shape, max_batch=2, max_seq=64, seed=5)
        toks[toks == 3] = 4
        model.embed[3] = float("nan") if spoil else 0.0
        cache, got = model.paged_cache(pages=16, page_size=16, max_seqs=4), []

        def spoiled():
            model.extend(cache, [2, 3], list(bad))
            assert model.logits.isnan().all() == spoil

        if captured:
            model.prefill(toks)
            model.capture()
        spoiled()
        model.extend(cache, [0, 1], list(toks))
        got.append(model.logits.clone())
        spoiled()
        model.prefill(toks)
        got.append(model.logits.clone())
        model.tokens.clamp_(min=4)
        spoiled()
        model.decode_step()
        got.append(model.logits.clone())
        return got

    for want, got in zip(run(False), run(True)):
        assert want.isfinite().all() and torch.equal(want, got)


def test_a_step_that_fails_is_as_if_it_had_not_been(kernels, monkeypatch):
    """A launch in the middle of a step is refused: the sequences are as long as before, and the step, taken again, gives
    what it gives in a run without the failure."""
    shape = LlamaShape(dim=256, n_heads=2, ffn=512, n_layers=2, vocab=512, block=64)
    model = LlamaU8(kernels, shape, max_batch=2, max_seq=64, seed=5)
    toks = list(torch.randint(0, shape.vocab, (2, 20), device="cuda", generator=gen(2)))
    steps = [([0, 1], [toks[0][:12], toks[1][:3]]), ([1, 0], [toks[1][3:], toks[0][12:]])]
    smooth, rough = (model.paged_cache(pages=8, page_size=16) for _ in range(2))
    want = []
    for seqs, t in steps:
        model.extend(smooth, seqs, t)
        want.append(model.logits.clone())
    real = kernels.attention_paged
    for (seqs, t), w in zip(steps, want):
        calls = []

        def second_fails(*a, **kw):
            calls.append(0)
            if len(calls) == 2:
                raise AdrError(4, "refused")
            return real(*a, **kw)

        before = ([list(p) for p in rough.pages], list(rough.length), sorted(rough.free))
        monkeypatch.setattr(kernels, "attention_paged", second_fails)
        with pytest.raises(AdrError):
            model.extend(rough, seqs, t)
        monkeypatch.setattr(kernels, "attention_paged", real)
        assert (rough.pages, rough.length, sorted(rough.free)) == before
        model.extend(rough, seqs, t)
        assert torch.equal(model.logits, w)
    kernels.device_status()
