"""What fails on the way leaves the paged cache and the harness as they were, and sizes that C's int does not hold are
refused.  No GPU: the kernels are a stand-in, on tensors of the host."""
from unittest import mock

import pytest
import torch

from adrastea_b200 import AdrError, RopeLayout, RopeTable, kernels as K
from adrastea_b200.llama import LlamaShape, LlamaU8, PagedCache


def state(c):
    return [list(p) for p in c.pages], list(c.length), list(c.free)


def model():
    shape = LlamaShape(dim=128, n_heads=2, ffn=64, n_layers=2, vocab=64, block=64)
    return LlamaU8(mock.MagicMock(), shape, max_batch=3, max_seq=64, device="cpu")


def test_a_table_that_cannot_be_written_leaves_the_cache_alone(monkeypatch):
    c = PagedCache(1, 8, 16, 1, 8, 3, 64, device="cpu")
    c.extend([0], [20])
    before, real, calls = state(c), torch.tensor, []

    def second_fails(*a, **kw):
        calls.append(0)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no memory")
        return real(*a, **kw)

    monkeypatch.setattr(torch, "tensor", second_fails)
    with pytest.raises(torch.OutOfMemoryError):
        c.extend([0, 1, 2], [20, 20, 20])
    monkeypatch.setattr(torch, "tensor", real)
    assert state(c) == before
    c.extend([0, 1, 2], [20, 20, 20])
    assert c.length == [40, 20, 20] and sorted(sum(c.pages, []) + c.free) == list(range(8))


@pytest.mark.parametrize("name", ["rms_norm", "matmul_nt_fp16u8", "rope_append_paged", "attention_paged",
                                  "attention_paged_workspace", "elementwise_binary_2d_f16"])
def test_a_step_that_fails_gives_its_positions_back(name):
    m = model()
    c = m.paged_cache(pages=9, page_size=16)
    toks = [torch.arange(20), torch.arange(3)]
    m.extend(c, [0, 2], toks)
    before = state(c)
    getattr(m.k, name).side_effect = AdrError(4, "refused")
    m._attention_ws = None
    with pytest.raises(AdrError):
        m.extend(c, [2, 0], [torch.arange(30), torch.arange(17)])
    assert state(c) == before
    getattr(m.k, name).side_effect = None
    m.extend(c, [2, 0], [torch.arange(30), torch.arange(17)])
    assert c.length == [37, 0, 33]


@pytest.mark.parametrize("tokens", [[torch.arange(20), torch.zeros(0, dtype=torch.int64)],   # none for the second
                                    [torch.arange(20), torch.tensor([64])],                  # no such row of the embedding
                                    [torch.arange(20)],                                      # one list too short
                                    [torch.arange(20), torch.arange(60)]])                   # more pages than there are
def test_tokens_that_are_refused_take_no_pages(tokens):
    m = model()
    c = m.paged_cache(pages=5, page_size=16)
    before = state(c)
    with pytest.raises((AssertionError, IndexError, MemoryError)):
        m.extend(c, [0, 1], tokens)
    assert state(c) == before


def test_truncated_sequences_give_back_the_pages_behind_their_end():
    c = PagedCache(1, 8, 4, 1, 8, 2, 32, device="cpu")
    c.extend([0, 1], [10, 3])
    c.truncate(0, 5)
    assert c.length == [5, 3] and len(c.pages[0]) == 2 and len(c.free) == 5
    c.truncate(0, 4)
    assert c.length[0] == 4 and len(c.pages[0]) == 1
    c.extend([0], [5])
    assert c.table[0, :3].tolist() == c.pages[0] and not set(c.pages[0]) & set(c.pages[1] + c.free)
    c.truncate(0, 0)
    assert c.pages[0] == [] and len(c.free) == 7
    for bad in (-1, 4):
        with pytest.raises(AssertionError):
            c.truncate(1, bad)
    with pytest.raises(AssertionError):
        c.truncate(2, 0)


def test_a_step_hands_over_as_much_of_the_table_as_it_needs():
    """The attention chooses its kernels by the table's width: a short batch in a cache for long sequences is a short one."""
    m = model()
    c = m.paged_cache(pages=9, page_size=16, max_positions=4096)
    for seqs, toks, columns in (([0], [20], 2), ([2, 0], [3, 13], 3), ([2], [13], 1), ([1, 2], [1, 1], 2)):
        m.extend(c, seqs, [torch.arange(n) for n in toks])
        for call in (m.k.rope_append_paged.call_args, m.k.attention_paged.call_args):
            table = next(a for a in call.args if torch.is_tensor(a) and a.dim() == 2 and a.dtype == torch.int32)
            assert table.is_contiguous() and torch.equal(table, c.table[seqs][:, :columns])


# ------------------------------------------------------------------ sizes
MANY = 1 << 32   # C's int would make 0 of it, and of MANY + 5 five


def rows(*dims):
    """Dimensions and the strides of a contiguous view."""
    s, strides = 1, []
    for d in reversed(dims):
        strides.append(s)
        s *= d
    return dims, tuple(reversed(strides))


@pytest.mark.parametrize("T,H", [(MANY + 5, 1), (1 << 31, 1), (2, MANY + 1)])
def test_rows_that_an_int_does_not_hold_are_refused(T, H):
    x, s = rows(T, H, 8)
    with pytest.raises(AssertionError):
        K._rope_plan(x, s, x, s, (T,))
    x, s = rows(T, H, 64)
    with pytest.raises(AssertionError):
        K._packed_plan(x, s, x, s, x, s, x, s, (3,))


@pytest.mark.parametrize("pages,sequences,columns", [(MANY + 5, 2, 4), (9, MANY + 2, 4), (9, 2, MANY + 4)])
def test_pages_and_tables_that_an_int_does_not_hold_are_refused(pages, sequences, columns):
    x, s = rows(6, 4, 64)
    kv, skv = rows(6, 2, 64)
    pool, sp = rows(pages, 16, 2, 64)
    tables = (sequences, columns), (sequences + 1,), (sequences,)
    with pytest.raises(AssertionError):
        K._append_plan(x, s, x, s, kv, skv, kv, skv, pool, sp, pool, sp, *tables)
    with pytest.raises(AssertionError):
        K._paged_plan(x, s, x, s, pool, sp, pool, sp, *tables)


def test_largest_rows_are_taken():
    T = (1 << 31) - 1
    x, s = rows(T, 1, 8)
    assert K._rope_plan(x, s, x, s, (T,))[:3] == (T, 1, 8)


@pytest.mark.parametrize("turns,rotary", [(torch.zeros(31, dtype=torch.int64), 64), (torch.zeros(64, dtype=torch.int64), 64),
                                          (torch.zeros((32, 1), dtype=torch.int64), 64), (torch.zeros(32), 64),
                                          (torch.zeros(32, dtype=torch.int64), 65)])
def test_a_table_of_another_size_is_refused(turns, rotary):
    """The kernels read rotary_dim / 2 numbers of it."""
    with pytest.raises((AssertionError, TypeError)):
        RopeTable(turns, rotary, RopeLayout.Half, 1.0)


def test_a_table_of_the_right_size_is_taken():
    assert RopeTable(torch.zeros(32, dtype=torch.int64), 64, RopeLayout.Half, 1.0).rotary_dim == 64


# ------------------------------------------------------------------ alignment
@pytest.mark.parametrize("name,change", [
    ("rope_f16", dict(out=1)), ("rope_f16", dict(inp=3)), ("rope_f16", dict(positions=2)), ("rope_f16", dict(turns=4)),
    ("rope_append_paged", dict(q_out=1)), ("rope_append_paged", dict(q=1)), ("rope_append_paged", dict(k=1)),
    ("rope_append_paged", dict(v=1)), ("rope_append_paged", dict(kp=1)), ("rope_append_paged", dict(vp=1)),
    ("rope_append_paged", dict(table=2)), ("rope_append_paged", dict(cu=1)), ("rope_append_paged", dict(lens=2)),
    ("rope_append_paged", dict(turns=4)), ("attention_packed", dict(cu=2)), ("attention_paged", dict(table=2)),
    ("attention_paged", dict(cu=2)), ("attention_paged", dict(lens=3))])
def test_pointers_between_elements_are_refused(name, change):
    """The GPU cannot read from there: the launch would end with a misaligned address."""
    from test_serving_host import CALLS, _lib, _ptr
    args = dict(CALLS[name], **{k: _ptr(offset) for k, offset in change.items()})
    assert getattr(_lib.load(), "adr_" + name)(*args.values()) == 2


@pytest.mark.parametrize("name", ["rope_f16", "rope_append_paged"])
def test_pointers_to_any_element_are_taken(name):
    """(As far as the missing context.)"""
    from test_serving_host import CALLS, _lib, _ptr
    halves = {"rope_f16": ("out", "inp"), "rope_append_paged": ("q_out", "q", "k", "v", "kp", "vp")}[name]
    args = dict(CALLS[name], **{k: _ptr(2) for k in halves})
    assert getattr(_lib.load(), "adr_" + name)(*args.values()) == 1
