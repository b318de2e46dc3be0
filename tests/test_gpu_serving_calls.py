"""Calls of the serving operators that the documentation allows: the captured and the concurrent ones with every output
checked against what went in, the largest sizes, arrays that contradict one another."""
import pytest
import torch

from adrastea_b200 import AdrError, RopeLayout, RopeScaling
from adrastea_b200.llama import LlamaShape, LlamaU8
from serving_oracle import assert_close, attend, positions_of, rotate
from test_gpu_serving import Pages, chain, gen, half, ints, paged_case, starts, view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pdl", [0, 1])
@pytest.mark.parametrize("m", [1, 2, 40])
def test_a_replayed_step_appends_what_it_is_given(kernels, pdl, m):
    """Lengths, the pages' order and the projections change between replays: the rotated queries, the slots that are written
    and all those that are not, and the attention follow what the arrays hold at the replay."""
    kernels.set_tunable("pdl", pdl)
    try:
        H, Hk, hd, page, n, most = 8, 2, 128, 16, 3, 1000
        g = gen(m)
        P = Pages(g, [most] * n, page, Hk, hd, fill=0.0)
        f16 = dict(dtype=torch.float16, device="cuda")
        st = dict(H=H, Hk=Hk, qkv=half(g, n * m, H + 2 * Hk, hd), q=torch.empty((n * m, H, hd), **f16), P=P,
                  cu=ints([i * m for i in range(n + 1)]), lens=ints([most] * n), rope=kernels.rope_table(hd, 10000.0), max_q=m,
                  scale=0.1, ws=kernels.attention_paged_workspace(H, Hk, hd), out=torch.empty((n * m, H, hd), **f16))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            chain(kernels, st)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain(kernels, st)
        for lens in ([100, 40, 1000], [m, 999, 64], [777, 50, 333]):
            order = torch.randperm(P.n, device="cuda", generator=g).to(torch.int32)
            P.table[:, :-1] = order[:n * (P.table.shape[1] - 1)].view(n, -1)
            P.k.copy_(half(g, *P.k.shape))
            P.v.copy_(half(g, *P.v.shape))
            st["lens"].copy_(ints(lens))
            st["qkv"].copy_(half(g, *st["qkv"].shape))
            st["q"].fill_(float("nan"))
            st["out"].fill_(float("nan"))
            want_v, want_k = P.v.clone(), P.k.double()
            tol_k = torch.zeros_like(want_k)
            graph.replay()
            torch.cuda.synchronize()
            kernels.device_status()
            q, k, v = st["qkv"].split([H, Hk, Hk], 1)
            for s in range(n):
                rows, pos = slice(s * m, (s + 1) * m), torch.arange(lens[s] - m, lens[s], device="cuda")
                assert_close(st["q"][rows], *rotate(q[rows], pos, hd, 10000.0, False, RopeScaling()), "q")
                at = P.table[s].long()[pos // page], pos % page
                want_k[at], tol_k[at] = rotate(k[rows], pos, hd, 10000.0, False, RopeScaling())
                want_v[at] = v[rows]
            assert_close(P.k, want_k, tol_k, "k")
            assert torch.equal(P.v, want_v)
            for s in range(n):
                keys, values = (positions_of(t, P.table[s], lens[s]) for t in (P.k, P.v))
                rows = slice(s * m, (s + 1) * m)
                assert_close(st["out"][rows], *attend(st["q"][rows], keys, values, 0.1, lens[s] - m + 1), s)
    finally:
        kernels.set_tunable("pdl", 0)


def test_many_calls_on_two_streams(kernels):
    """Both streams are kept busy, with a workspace each and an output for each call: every one of them is right."""
    jobs = []
    for i, (H, Hk, hd, new, lens) in enumerate([(32, 8, 128, [1] * 6, [3000, 10, 500, 1500, 64, 2000]),
                                                (16, 16, 64, [40, 1, 9], [2500, 700, 9])]):
        q, P, kv, cu = paged_case(new, lens, H, Hk, hd, 32, "tokens", seed=i, spare=0)
        outs = [torch.full_like(q, float("nan")) for _ in range(12)]
        jobs.append((torch.cuda.Stream(), q, P, kv, new, lens, ints(cu), ints(lens), outs,
                     kernels.attention_paged_workspace(H, Hk, hd)))
    torch.cuda.synchronize()
    for r in range(12):
        for stream, q, P, kv, new, lens, cu, n, outs, ws in jobs:
            kernels.attention_paged(view(outs[r]), view(q), P.k, P.v, P.table, cu, n, max(new), 0.1, ws, stream=stream)
    torch.cuda.synchronize()
    kernels.device_status()
    for stream, q, P, kv, new, lens, cu, n, outs, ws in jobs:
        at = starts(new)
        for s in range(len(new)):
            rows = slice(at[s], at[s + 1])
            assert_close(outs[0][rows], *attend(q[rows], *kv[s], 0.1, lens[s] - new[s] + 1), s)
        assert all(torch.equal(outs[0], o) for o in outs[1:])


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


@pytest.mark.parametrize("H,Hk,hd", [(8, 2, 96), (8, 3, 64), (130, 2, 64), (0, 1, 64), (4, -1, 64)])
def test_a_workspace_of_heads_that_are_not_taken_is_refused(kernels, H, Hk, hd):
    with pytest.raises(AdrError) as e:
        kernels.attention_paged_workspace(H, Hk, hd)
    assert e.value.code == 2
