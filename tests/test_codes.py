"""The tests' own account of the 8-bit cache against torch's cast, on the CPU."""
import torch

from codes import HIGH, LOW, MOST, E4M3, code_of, exponent, held, values


def every_half():
    x = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.float16)
    return x[x.isfinite()].double()


def test_exponents():
    e = torch.arange(LOW, HIGH + 1)
    top = 448.0 * 2.0 ** e.double()
    assert torch.equal(exponent(top[:-1]), e[:-1].int())
    up = torch.nextafter(top.float(), torch.tensor(float("inf"))).double()
    assert torch.equal(exponent(up[:-1]), (e[:-1] + 1).int())
    assert exponent(torch.tensor([0.0, 65504.0, 57344.0, 57376.0], dtype=torch.float64)).tolist() \
        == [LOW, HIGH, HIGH - 1, HIGH]


def test_codes_are_torchs():
    x = every_half()
    for e in range(LOW, HIGH + 1):
        y = x[(x.abs() <= 448.0 * 2.0 ** e) & (x.abs() <= MOST)]
        ref = (y / 2.0 ** e).float().to(E4M3)
        h = held(y, torch.tensor(e))
        assert torch.equal(h, ref.float().double() * 2.0 ** e)
        n = h.numel()
        c = code_of(h.view(1, 1, 1, 1, n), torch.full((1, 1, 1), e))
        assert torch.equal(c.flatten(), ref.view(torch.uint8))
        back = values(c, torch.full((1, 1, 1), e)).flatten()
        assert torch.equal(back, h) and torch.equal(h.half().double(), h)  # fp16 numbers


def test_error_of_a_code():
    """Half a step of four bits, 2^-4, or half of 2^(e - 9)."""
    x = every_half()
    for e in (LOW, -3, HIGH):
        y = x[x.abs() <= 448.0 * 2.0 ** e]
        d = (held(y, torch.tensor(e)) - y).abs()
        assert bool((d <= torch.clamp(y.abs() * 2.0 ** -4, min=2.0 ** (e - 10))).all())


def test_not_finite():
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0], dtype=torch.float64)
    h = held(x, torch.tensor(0))
    assert h.isnan().tolist() == [True, True, True, False]
    c = code_of(h.view(1, 1, 1, 1, 4), torch.zeros(1, 1, 1))
    assert (c.flatten() & 0x7F)[:3].tolist() == [0x7F] * 3
