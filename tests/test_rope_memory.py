"""What rope_cache_write's ``out`` may share with q, k and v, without a GPU."""

import numpy as np
import pytest
import torch

from test_native_calls_added import FUNCTIONS, native  # noqa: F401  (the fixture)


@pytest.fixture(scope="module")
def C():
    from femtovllm import _C

    return _C


def packed(tokens, *heads, dim=8):
    """Columns of one (tokens, sum(heads) * dim) array, as a fused projection leaves q, k and v."""
    x = torch.zeros(tokens, sum(heads), dim, dtype=torch.bfloat16)
    return x.split(list(heads), dim=1)


def test_share_elements(C):
    q, k, v = packed(5, 4, 2, 2)
    assert not C._share_elements(q, k) and not C._share_elements(k, v) and not C._share_elements(v, q)
    assert C._share_elements(q, q) and C._share_elements(q, q[2:3]) and C._share_elements(q[:, 3:], q)
    assert not C._share_elements(q[:2], q[2:]) and not C._share_elements(q, torch.zeros_like(q))
    x = torch.zeros(6, 4, 3, 8)
    assert not C._share_elements(x[:, :, 0], x[:, :, 2])  # heads of q, k and v in turn
    assert C._share_elements(x[:, :, 0], x[:3].reshape(9, 4, 8))  # other strides
    y = torch.zeros(400)
    for off, shared in ((0, True), (7, True), (8, False), (16, False), (23, False), (24, False), (25, True)):
        # rows of 8 at 0, 32, 64, ..; other rows of 8 from `off` on
        assert C._share_elements(y.as_strided((3, 2, 8), (64, 32, 1)), y[off:].as_strided((3, 2, 8), (64, 32, 1))) == shared, off
    assert not C._share_elements(q[:0], q)


def test_share_elements_against_sets(C):
    rng = np.random.default_rng(0)
    found = [0, 0]
    for _ in range(400):
        views, sets = [], []
        x = torch.zeros(600)
        for _ in range(2):
            t, h, s0, s1, off = (int(rng.integers(*r)) for r in ((1, 5), (1, 5), (0, 60), (0, 60), (0, 60)))
            views.append(x[off:].as_strided((t, h, 4), (s0, s1, 1)))
            sets.append({off + i * s0 + j * s1 + d for i in range(t) for j in range(h) for d in range(4)})
        want = bool(sets[0] & sets[1])
        assert C._share_elements(*views) == want
        found[want] += 1
    assert min(found) > 20


@pytest.mark.parametrize("case,taken", [("own", True), ("columns", True), ("k is q", False), ("v is q", False),
                                        ("k ahead by a token", False), ("heads in turn", False)])
def test_native_call_in_place(native, case, taken):  # noqa: F811
    """out is q: taken where q plainly holds no element of k and v, else left to the Python path, which looks closer."""
    module, counts = native[:2]
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    pool, tab = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(64, 64)
    q, k, v = (torch.zeros(3, h, 128, dtype=torch.bfloat16) for h in (4, 2, 2))
    if case == "columns":
        q, k, v = packed(3, 4, 2, 2, dim=128)
    elif case == "k is q":
        k = q[:, :2]
    elif case == "v is q":
        v = q[:, 2:]
    elif case == "k ahead by a token":
        x = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
        q, k = x[:3], x[1:, :2]
    elif case == "heads in turn":
        x = torch.zeros(3, 2, 3, 128, dtype=torch.bfloat16)
        q, k, v = x.unbind(2)
    before = counts.get(FUNCTIONS[3], 0)
    out = module.rope(q, k, v, tab, tab, i32(3), pool, pool, i32(3, 2), None, 1, False, q)
    assert (out is not None) == taken and counts.get(FUNCTIONS[3], 0) == before + taken


def test_rows_meet(C):
    q, k, v = packed(5, 4, 2, 2)
    x = torch.zeros(400)
    assert not C._rows_meet(q) and not C._rows_meet(k[:1]) and not C._rows_meet(q[:0])
    assert not C._rows_meet(torch.zeros(4, 5, 8).transpose(0, 1))
    assert C._rows_meet(q[:1].expand(5, -1, -1)) and C._rows_meet(q[:, :1].expand(-1, 4, -1))
    assert not C._rows_meet(q[:1, :1].expand(1, 1, -1))
    assert C._rows_meet(x.as_strided((3, 2, 8), (15, 8, 1))) and not C._rows_meet(x.as_strided((3, 2, 8), (16, 8, 1)))


@pytest.mark.parametrize("strides,taken", [((512, 128), True), ((0, 128), False), ((512, 0), False), ((511, 128), False),
                                           ((640, 128), True), ((128, 384), False)])
def test_native_call_with_rows_that_meet(native, strides, taken):  # noqa: F811
    """In place, q's rows plainly apart; the others, the heads ahead of the tokens among them, go to the Python path."""
    module, counts = native[:2]
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    b16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    pool, tab = b16(4, 2, 16, 128), torch.zeros(64, 64)
    q = b16(4000).as_strided((3, 4, 128), (*strides, 1))
    before = counts.get(FUNCTIONS[3], 0)
    out = module.rope(q, b16(3, 2, 128), b16(3, 2, 128), tab, tab, i32(3), pool, pool, i32(3, 2), None, 1, False, q)
    assert (out is not None) == taken and counts.get(FUNCTIONS[3], 0) == before + taken
