"""Host side of the operators over sequences of different lengths: the rotation's table and the refusals.  No GPU."""
import ctypes as C
import math

import pytest

from adrastea_b200 import AdrError, RopeScaling, _lib, rope_turns
from adrastea_b200.build import build_library
from serving_oracle import frequencies

build_library()

SCALINGS = [RopeScaling.Identity(), RopeScaling.Linear(4), RopeScaling.Base(8), RopeScaling.Bands(8, 8192),
            RopeScaling.Bands(2, 100, 0.5, 40), RopeScaling.Yarn(16, 4096), RopeScaling.Yarn(1, 2048),
            RopeScaling.Yarn(4, 64, 2.0, 1.0)]


@pytest.mark.parametrize("d", [2, 8, 50, 64, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 1.5])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_turns_are_the_frequencies(d, theta, scaling):
    if scaling.kind == 2 and d < 4:
        return
    turns, amplitude = rope_turns(d, theta, scaling)
    want, amp = frequencies(d, theta, scaling)
    assert len(turns) == d // 2
    # the oracle's 64-bit arithmetic: some ten roundings of 2^-53, the power's exponent of up to ln(theta) * 1
    for t, f in zip(turns, want):
        assert abs(t / 2.0 ** 64 * 2 * math.pi - f) <= 2.0 ** -48 * f + 2.0 ** -61
    assert abs(amplitude - amp) <= 2.0 ** -24 * amp


def test_far_positions_keep_their_angle():
    """position * turns modulo 2^64 against the angle in 200-bit integers: off by position * 2^-64 turns at most."""
    turns, _ = rope_turns(128, 10000.0)
    f = turns[0]
    # pair 0 turns by one radian per position: 2^64 / (2 pi), from a 60-digit pi
    pi = 314159265358979323846264338327950288419716939937510582097494
    exact = (10 ** 59 << 64) // (2 * pi)
    assert abs(f - exact) <= 1
    for p in (1, 131071, 1 << 20, (1 << 31) - 1, -5, -(1 << 31)):
        got = (p * f) % (1 << 64)
        want = ((p * 10 ** 59 << 64) // (2 * pi)) % (1 << 64)
        assert min((got - want) % (1 << 64), (want - got) % (1 << 64)) <= abs(p) + 1


@pytest.mark.parametrize("args,code", [((7, 1e4, 0, 1, 0, 0, 0), 2), ((0, 1e4, 0, 1, 0, 0, 0), 1),
                                       ((64, 1.0, 0, 1, 0, 0, 0), 1), ((64, float("nan"), 0, 1, 0, 0, 0), 1),
                                       ((64, float("inf"), 0, 1, 0, 0, 0), 1), ((64, 1e4, 5, 1, 0, 0, 0), 1),
                                       ((64, 1e4, 1, 0.5, 0, 0, 0), 1), ((64, 1e4, 1, float("nan"), 0, 0, 0), 1),
                                       ((2, 1e4, 2, 2, 0, 0, 0), 2), ((64, 1e4, 3, 2, 0, 1, 4), 1),
                                       ((64, 1e4, 3, 2, 4096, 4, 4), 1), ((64, 1e4, 4, 2, 4096, 0, 32), 1)])
def test_turns_refuse(args, code):
    d, theta, kind, *rest = args
    with pytest.raises(AdrError) as e:
        rope_turns(d, theta, RopeScaling(kind, *rest))
    assert e.value.code == code


def _ll(*v):
    return (C.c_longlong * len(v))(*v)


def _ptr(offset=0):
    return C.c_void_p(0x10000 + offset)


ROPE = dict(ctx=None, stream=None, out=_ptr(), inp=_ptr(), tokens=3, heads=4, hd=64, so=_ll(256, 64), si=_ll(256, 64),
            positions=_ptr(), turns=_ptr(), rotary=64, amplitude=1.0, layout=0)
APPEND = dict(ctx=None, stream=None, q_out=_ptr(), q=_ptr(), k=_ptr(), v=_ptr(), kp=_ptr(), vp=_ptr(), tokens=3, n=2,
              heads=4, kv=2, hd=64, sqo=_ll(256, 64), sq=_ll(256, 64), sk=_ll(128, 64), sv=_ll(128, 64),
              skp=_ll(2048, 128, 64), svp=_ll(2048, 128, 64), table=_ptr(), cu=_ptr(), lens=_ptr(), max_pages=4,
              page=16, pages=9, turns=_ptr(), rotary=64, amplitude=1.0, layout=1)
PACKED = dict(ctx=None, stream=None, out=_ptr(), q=_ptr(), k=_ptr(), v=_ptr(), tokens=3, n=2, max_q=2, heads=4, kv=2,
              hd=64, so=_ll(256, 64), sq=_ll(256, 64), sk=_ll(128, 64), sv=_ll(128, 64), cu=_ptr(), scale=0.125, mask=1)
PAGED = dict(ctx=None, stream=None, out=_ptr(), q=_ptr(), kp=_ptr(), vp=_ptr(), tokens=3, n=2, max_q=2, heads=4, kv=2,
             hd=64, so=_ll(256, 64), sq=_ll(256, 64), skp=_ll(2048, 128, 64), svp=_ll(2048, 128, 64), table=_ptr(),
             cu=_ptr(), lens=_ptr(), max_pages=4, page=16, pages=9, scale=0.125, ws=_ptr(), bytes=1 << 40)
CALLS = {"rope_f16": ROPE, "rope_append_paged": APPEND, "attention_packed": PACKED, "attention_paged": PAGED}
# what is wrong, the answer.  1: invalid, 2: a shape, stride or alignment that is not taken.
BAD = [("rope_f16", dict(out=None), 1), ("rope_f16", dict(positions=None), 1), ("rope_f16", dict(turns=None), 1),
       ("rope_f16", dict(tokens=0), 1), ("rope_f16", dict(heads=-1), 1), ("rope_f16", dict(rotary=63), 2),
       ("rope_f16", dict(rotary=66), 2), ("rope_f16", dict(hd=264, rotary=64), 2), ("rope_f16", dict(layout=2), 1),
       ("rope_f16", dict(amplitude=float("nan")), 1), ("rope_f16", dict(so=None), 1), ("rope_f16", dict(si=_ll(-1, 64)), 1),
       ("rope_append_paged", dict(v=None), 1), ("rope_append_paged", dict(table=None), 1),
       ("rope_append_paged", dict(n=0), 1), ("rope_append_paged", dict(page=0), 1), ("rope_append_paged", dict(pages=0), 1),
       ("rope_append_paged", dict(max_pages=-1), 1), ("rope_append_paged", dict(skp=_ll(1, -1, 1)), 1),
       ("rope_append_paged", dict(rotary=0), 1), ("rope_append_paged", dict(hd=258, rotary=64), 2),
       ("attention_packed", dict(k=None), 1), ("attention_packed", dict(cu=None), 1), ("attention_packed", dict(n=0), 1),
       ("attention_packed", dict(max_q=0), 1), ("attention_packed", dict(mask=2), 1),
       ("attention_packed", dict(scale=float("inf")), 1), ("attention_packed", dict(hd=80), 2),
       ("attention_packed", dict(heads=5), 2), ("attention_packed", dict(heads=130, kv=2), 2),
       ("attention_packed", dict(sq=_ll(260, 64)), 2), ("attention_packed", dict(sk=_ll(128, 36)), 2),
       ("attention_packed", dict(so=_ll(256, 0)), 2), ("attention_packed", dict(sv=_ll(-128, 64)), 1),
       ("attention_packed", dict(q=_ptr(2)), 2), ("attention_packed", dict(out=_ptr(8)), 2),
       ("attention_paged", dict(ws=None), 1), ("attention_paged", dict(lens=None), 1), ("attention_paged", dict(page=24), 2),
       ("attention_paged", dict(page=8), 2), ("attention_paged", dict(page=512), 2), ("attention_paged", dict(pages=0), 1),
       ("attention_paged", dict(hd=96), 2), ("attention_paged", dict(heads=3), 2), ("attention_paged", dict(ws=_ptr(4)), 2),
       ("attention_paged", dict(skp=_ll(2048, 130, 64)), 2), ("attention_paged", dict(svp=_ll(2048, 128, 0)), 2),
       ("attention_paged", dict(max_pages=1 << 27), 2), ("attention_paged", dict(kp=_ptr(2)), 2)]


@pytest.mark.parametrize("name,change,code", BAD)
def test_entry_points_refuse_before_touching_a_gpu(name, change, code):
    """Arguments are looked at before the context: without one, a wrong call says what is wrong with it."""
    args = dict(CALLS[name], **change)
    assert getattr(_lib.load(), "adr_" + name)(*args.values()) == code


@pytest.mark.parametrize("name", CALLS)
def test_a_right_call_without_a_context_is_refused(name):
    assert getattr(_lib.load(), "adr_" + name)(*CALLS[name].values()) == 1


@pytest.mark.parametrize("change", [dict(sq=_ll(3, 64), tokens=1), dict(sk=_ll(128, 7), kv=1, heads=4)])
def test_strides_of_single_rows_and_heads_do_not_matter(change):
    """A dimension of one element has no stride to speak of: such a call gets as far as the missing context."""
    assert _lib.load().adr_attention_packed(*dict(PACKED, **change).values()) == 1


def test_workspace_of_no_context_is_nothing():
    assert _lib.load().adr_attention_paged_workspace(None, 32, 8, 128) == 0
