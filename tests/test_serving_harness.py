"""Sequences of different lengths through the LLaMA-shape harness over a paged cache (`LlamaU8.extend`), against
recomputation of every prefix, and the cache's bookkeeping (which needs no GPU)."""
import pytest
import torch

from adrastea_b200.llama import LlamaShape, LlamaU8, PagedCache


def cache(pages=6, page_size=4, max_seqs=3, max_positions=16):
    return PagedCache(1, pages, page_size, 1, 8, max_seqs, max_positions, device="cpu")


def test_pages_are_handed_out_as_sequences_grow():
    c = cache()
    c.extend([0, 2], [5, 4])
    assert [len(p) for p in c.pages] == [2, 0, 1] and c.length == [5, 0, 4]
    c.extend([0, 2], [3, 1])          # the first still fits, the second starts a page
    assert [len(p) for p in c.pages] == [2, 0, 2] and len(c.free) == 2
    used = c.pages[0] + c.pages[2]
    assert len(set(used)) == 4 and not set(used) & set(c.free)
    assert c.table[0, :2].tolist() == c.pages[0] and c.table[2, :2].tolist() == c.pages[2]
    assert (c.table[1] == -1).all() and (c.table[:, 2:] == -1).all()
    c.extend([1], [0])
    assert c.pages[1] == []


def test_a_refused_extension_changes_nothing():
    c = cache()
    c.extend([0], [15])
    before = (list(c.free), [list(p) for p in c.pages], list(c.length), c.table.clone())
    for seqs, new in (([0, 1], [1, 9]), ([1], [17]), ([0], [2])):   # no pages, past the table's row
        with pytest.raises(MemoryError):
            c.extend(seqs, new)
        assert (c.free, c.pages, c.length) == before[:3] and torch.equal(c.table, before[3])
    with pytest.raises(AssertionError):
        c.extend([1, 1], [1, 1])


def test_released_pages_come_back():
    c = cache()
    c.extend([0, 1], [16, 8])
    assert c.free == []
    c.release(0)
    assert len(c.free) == 4 and c.length[0] == 0
    c.extend([2], [16])
    assert sorted(c.pages[2] + c.pages[1]) == list(range(6))


@pytest.mark.gpu
@pytest.mark.parametrize("n_heads,page_size", [(4, 16), (2, 64)])  # head_dim 64 and 128
def test_prompts_chunks_and_tokens_in_one_batch(kernels, n_heads, page_size):
    """Two sequences grow by prompts, chunks and tokens, a third joins and one leaves; after every step the logits
    are those of the whole prefix (the harness's own tolerance for its fp16 chain)."""
    from test_llama_harness import ref_forward
    g = torch.Generator(device="cuda").manual_seed(n_heads)
    shape = LlamaShape(dim=256, n_heads=n_heads, ffn=512, n_layers=2, vocab=512, block=64)
    model = LlamaU8(kernels, shape, max_batch=3, max_seq=320, seed=3)
    model.embed.mul_(0.5)
    cache = model.paged_cache(pages=3 * 320 // page_size - 2, page_size=page_size)
    draw = lambda n: torch.randint(0, shape.vocab, (n,), device="cuda", generator=g)
    hist = {}

    def step(**new):
        seqs = [int(s[1:]) for s in new]
        toks = [draw(n) for n in new.values()]
        for s, t in zip(seqs, toks):
            hist[s] = torch.cat([hist[s], t]) if s in hist else t
        got = model.extend(cache, seqs, toks)
        kernels.device_status()
        for i, s in enumerate(seqs):
            want = ref_forward(model, kernels, hist[s][None])
            rel = ((model.logits[i].float() - want[0].float()).abs().max() / want.float().abs().max()).item()
            assert rel < 3e-2, (s, rel)
            assert got[i] == model.logits[i].argmax()

    step(s0=12, s1=150)
    step(s0=1, s1=1)
    step(s1=70, s0=1)
    step(s2=30, s0=40, s1=1)
    step(s0=1, s1=1, s2=1)
    cache.release(1)
    del hist[1]
    step(s1=200, s2=1)
    step(s0=1, s1=1, s2=1)


@pytest.mark.gpu
def test_extend_agrees_with_prefill_and_decode(kernels):
    """Prompts of one length, then tokens: what the rectangular cache gives (both within the tolerance of their chain)."""
    shape = LlamaShape(dim=256, n_heads=2, ffn=512, n_layers=2, vocab=512, block=64)
    model = LlamaU8(kernels, shape, max_batch=2, max_seq=64, seed=5)
    model.embed.mul_(0.5)
    toks = torch.randint(0, shape.vocab, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    cache = model.paged_cache(pages=8, page_size=16)
    model.prefill(toks)
    want = model.logits.clone()
    model.extend(cache, [0, 1], list(toks))
    assert (model.logits - want).abs().max() < 3e-2 * want.abs().max()
    nxt = model.tokens.clone()
    model.decode_step()
    want = model.logits.clone()
    model.extend(cache, [1, 0], [nxt[1:], nxt[:1]])
    assert (model.logits.flip(0) - want).abs().max() < 3e-2 * want.abs().max()
    kernels.device_status()
