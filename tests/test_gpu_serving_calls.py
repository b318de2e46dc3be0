"""Calls of the serving operators that the documentation allows: the captured and the concurrent ones with every output
checked against what went in, the largest sizes, arrays that contradict one another."""
import pytest
import torch

from adrastea_b200 import AdrError, RopeLayout, RopeScaling
from adrastea_b200.llama import LlamaShape, LlamaU8
from serving_oracle import assert_close, attend, positions_of, rotate
from test_gpu_serving import Pages, chain, gen, half, ints, paged_case, starts, view

pytestmark = pytest.mark.gpu


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
