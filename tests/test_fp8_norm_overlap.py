"""fp8.add_rmsnorm refuses results among its operands (before the device is looked at, so no GPU is needed): a row's group
would read what another has written already.  What is laid side by side, or is an operand itself, passes this check, and works."""
import itertools

import pytest
import torch

from tierlm_amd import fp8

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
T, n = 5, 40


def rows(flat, at, stride, count=T, width=n):
    return flat.as_strided((count, width), (stride, 1), at)


def refused(match, *a, **kw):
    with pytest.raises(ValueError, match=match):
        fp8.add_rmsnorm(*a, **kw)


@pytest.fixture
def w():
    return torch.ones(n)


def test_shifted_places(w):
    """By a value, a row and the whole span, to either side, with and without gaps."""
    flat = torch.zeros(2000)
    for stride in (n, n + 9):
        span = (T - 1) * stride + n
        for shift, match in ((1, "overlap"), (n - 1, "overlap"), (stride, "overlap"), (stride + 3, "overlap"),
                             (span - 1, "overlap"), (span, "device"), (span + 7, "device")):
            for a, b in ((0, shift), (shift, 0)):
                h, o = rows(flat, a, stride), rows(flat, b, stride)
                refused(match, h, None, w, out=o)
                refused(match, h, torch.zeros(T, n), w, out=o)
                refused(match, torch.zeros(T, n), h, w, out=o)     # over x
                refused(match, h, o, w)                             # in place, x shifted


def test_operands_themselves(w):
    h, x = torch.zeros(T, n), torch.zeros(T, n)
    for a in ((h, x, w), (h, h, w), (h, None, w)):
        refused("device", *a)
    for a, o in ((h, h), (h, x), (x, h), (h, torch.zeros(T, n))):
        refused("device", a, x, w, out=o)
    refused("device", h.half(), None, w)
    one = torch.zeros(400)                                          # one row: strides say nothing
    refused("device", rows(one, 3, 50, 1), rows(one, 3, 90, 1), w, out=rows(one, 3, n, 1))
    refused("overlap", rows(one, 3, 50, 1), None, w, out=rows(one, 4, 50, 1))
    # the same address, rows further apart
    flat = torch.zeros(1000)
    refused("overlap", rows(flat, 0, n), None, w, out=rows(flat, 0, n + 1))
    refused("overlap", rows(flat, 0, n), rows(flat, 0, n + 8), w)


def test_side_by_side(w):
    """Columns of one wider buffer, and rows between rows."""
    flat = torch.zeros(3000)
    for gap in (0, 5):
        stride = 2 * n + 2 * gap
        a, b = rows(flat, 0, stride), rows(flat, n + gap, stride)
        for h, o in ((a, b), (b, a)):
            refused("device", h, None, w, out=o)
            refused("device", h, o, w)
            refused("device", torch.zeros(T, n), h, w, out=o)
    refused("overlap", rows(flat, 0, 2 * n), rows(flat, n + 1, 2 * n), w)      # its last value is the next row's first
    refused("overlap", rows(flat, 0, 2 * n), rows(flat, n - 1, 2 * n), w)
    # rows of another stride, and of another type, in the gaps
    refused("device", rows(flat, 0, 3 * n), rows(flat, 2 * n, 6 * n), w)
    half = flat.view(F16)
    refused("device", rows(flat, 0, 2 * n), rows(half, 2 * n, 4 * n), w)       # 2 n bytes inside the gap of 4 n
    refused("overlap", rows(flat, 0, 2 * n), rows(half, 2 * n - 1, 4 * n), w)
    refused("overlap", rows(flat, 0, 2 * n), rows(half, 2 * n, 3 * n), w)


def test_codes_and_scale_and_weights(w):
    flat = torch.zeros(4000)
    bytes8 = flat.view(torch.uint8).view(torch.float8_e4m3fn)
    h, x = rows(flat, 0, n), rows(flat, 1000, n)
    codes = lambda at: bytes8[at:at + T * 128].view(T, 128)        # noqa: E731
    scale = lambda at: flat[at:at + T].view(T, 1)                  # noqa: E731
    for at, match in ((0, "overlap"), (4 * T * n - 1, "overlap"), (4 * T * n, "device"), (4000 - T * 128 + 1, "overlap"),
                      (4000 - T * 128, "device"), (4000 + 4 * T * n - 1, "overlap")):
        refused(match, h, x, w, codes=codes(at))
    for at, match in ((T * n - 1, "overlap"), (T * n, "device"), (1000 - T, "device"), (1001 - T, "overlap")):
        refused(match, h, x, w, scale=scale(at))
        refused(match, h, x, w, out=rows(flat, 2000, n), scale=scale(at))
    refused("overlap", h, x, w, out=rows(flat, 2000, n), scale=scale(2003))
    refused("overlap", h, x, w, codes=codes(8000), scale=scale(2000))
    refused("device", h, x, w, codes=codes(8000), scale=scale(2000 + T * 32))
    wf = flat[3000:3000 + n]
    refused("overlap", h, x, wf, out=rows(flat, 3000 + n - 1, n))
    refused("overlap", h, x, wf, scale=scale(3000))
    refused("overlap", h[:1], None, wf, out=wf.view(1, n))         # the weights' own place: they are read after it is written
    refused("overlap", wf.view(1, n), h[:1], wf)
    refused("device", wf.view(1, n), None, wf)                     # nothing is stored there


def test_every_pair_of_rows():
    """The test of two sets of rows against one of all their bytes."""
    for (pa, sa, wa, na), (pb, sb, wb, nb) in itertools.product(
            itertools.product((0, 3), (5, 8), (1, 5), (1, 3)), itertools.product(range(0, 30, 1), (4, 5, 8, 11), (1, 4), (0, 1, 2, 3))):
        one = {pa + i * sa + j for i in range(na) for j in range(wa)}
        two = {pb + i * sb + j for i in range(nb) for j in range(wb)}
        assert fp8._rows_meet((pa, sa, wa, na), (pb, sb, wb, nb)) == bool(one & two)
        assert fp8._rows_meet((pb, sb, wb, nb), (pa, sa, wa, na)) == bool(one & two)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [40, 3000, 9001])
def test_what_passes_works(hip, width):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    h0, x0 = (torch.randn(T, width, generator=g, device="cuda") for _ in range(2))
    w = 1 + 0.1 * torch.randn(width, generator=g, device="cuda")
    want_h = h0.clone()
    want = fp8.add_rmsnorm(want_h, x0.clone(), w)

    def check(got, sums):
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
        assert torch.equal(sums, want_h)

    h, x = h0.clone(), x0.clone()
    check(fp8.add_rmsnorm(h, x, w, out=x), x)                      # over x
    assert torch.equal(h, h0)
    both = torch.stack([h0, x0], 1).reshape(2 * T, width)          # rows between rows
    check(fp8.add_rmsnorm(both[0::2], both[1::2], w), both[0::2])
    assert torch.equal(both[1::2], x0)
    cols = torch.cat([h0, x0], 1)
    check(fp8.add_rmsnorm(cols[:, :width], cols[:, width:], w, out=cols[:, width:]), cols[:, width:])
    twice = fp8.add_rmsnorm(h, h, w)                               # x is h
    assert torch.equal(h, h0 + h0)
    again = fp8.add_rmsnorm(h, None, w)
    assert torch.equal(twice[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(twice[1], again[1])
