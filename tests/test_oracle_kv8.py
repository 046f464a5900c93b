"""The 8-bit cache's definition (``oracle/kv8.py``) on the CPU: the scale rule, the error bounds that the
format promises, and the growth of a page's scale."""

from __future__ import annotations

import math

import pytest
import torch

from oracle.kv8 import EXPONENTS, Kv8Cache, exponent


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_value_is_a_number_of_the_type(dtype):
    for e in EXPONENTS[dtype]:
        for q in (1, 63, 127):
            v = torch.tensor(math.ldexp(q, e), dtype=torch.float64)
            assert v.to(dtype).double() == v and torch.isfinite(v.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_exponent_is_the_smallest_that_holds(dtype):
    lo, hi = EXPONENTS[dtype]
    g = torch.Generator().manual_seed(0)
    top = float(torch.finfo(dtype).max)
    amax = [0.0, top, top / 2, 127.0, 127.5, 127.25, 128.0, 1.0, 1e-7, 255.0, 254.9]
    amax += torch.randn(200, generator=g).abs().to(dtype).tolist()
    for a in amax:
        a = float(torch.tensor(a).to(dtype))
        e = exponent(a, dtype)
        assert lo <= e <= hi
        if e > lo:
            assert round(math.ldexp(a, 1 - e)) > 127
        if e < hi:
            assert round(math.ldexp(a, -e)) <= 127
    assert exponent(float("inf"), dtype) == exponent(float("nan"), dtype) == "nan"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs", [4, 16, 32])
def test_error_bounds_of_a_write_and_of_appends(dtype, bs):
    """At most half a step when a page is written at once; less than one step of its last scale when it
    was filled token by token, however often the scale grew."""
    g = torch.Generator().manual_seed(bs)
    d = 8
    x = (torch.randn(1, 1, bs, d, generator=g) * torch.logspace(-2, 2, bs)[:, None]).to(dtype)
    tables = torch.tensor([[0]])
    once, many = (Kv8Cache(1, 1, bs, d, dtype) for _ in range(2))
    once.write(tables, [0], x, x)
    for t in range(bs):
        many.write(tables, [t], x[:, :, t:t + 1], x[:, :, t:t + 1])
    step = 2.0 ** once.exps[0, 0, 0]
    assert many.exps[0, 0, 0] == once.exps[0, 0, 0]
    assert (once.values(0, 0, 0) - x[0, 0].double()).abs().max() <= step / 2
    assert (many.values(0, 0, 0) - x[0, 0].double()).abs().max() < step


def test_a_write_at_slot_zero_starts_the_page_anew_and_one_inside_keeps():
    c = Kv8Cache(1, 1, 4, 8, torch.float16)
    t = torch.tensor([[0]])
    big, small = torch.full((1, 1, 2, 8), 1000.0).half(), torch.full((1, 1, 1, 8), 0.5).half()
    c.write(t, [0], big, big)
    c.write(t, [2], small, small)
    assert c.exps[0, 0, 0] == 3 and torch.equal(c.values(0, 0, 0)[:2], torch.full((2, 8), 1000.0).double())
    assert (c.values(0, 0, 0)[2] == 0).all()  # 0.5 / 8 rounds to 0 beside 1000
    c.write(t, [0], small, small)
    assert c.exps[0, 0, 0] == -7 and (c.values(0, 0, 0)[0] == 0.5).all()


def test_values_that_are_not_finite_poison_their_page_until_it_starts_anew():
    c = Kv8Cache(2, 1, 4, 8, torch.float16)
    t = torch.tensor([[0, 1]])
    x = torch.ones(1, 1, 5, 8).half()
    x[0, 0, 1, 3] = float("inf")
    c.write(t, [0], x, x)
    assert torch.isnan(c.values(0, 0, 0)).all() and torch.isfinite(c.values(1, 0, 0)).all()
    c.write(t, [2], x[:, :, :1], x[:, :, :1])
    assert torch.isnan(c.values(0, 0, 0)).all()
    c.write(t, [0], x[:, :, :1], x[:, :, :1])
    assert torch.isfinite(c.values(0, 0, 0)).all()
