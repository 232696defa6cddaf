"""What the attention over the E4M3 cache takes for granted about its weights' terms."""
import torch


def test_three_e5m2_terms_are_a_half():
    """Every half up to 2^15 is t + t' / 16 + t'' / 256 with E5M2 numbers, each the nearest to what is left, and 16 times the rest never leaves the type's range."""
    x = torch.arange(0x7801, dtype=torch.int32).to(torch.int16).view(torch.float16)      # 0, 2^-24, ... 2^15
    assert x[-1] == 2.0 ** 15 and x[1] == 2.0 ** -24
    total, rest, unit = torch.zeros(len(x), dtype=torch.float64), x, 1.0
    for _ in range(3):
        term = rest.to(torch.float8_e5m2).to(torch.float16)
        total += term.double() * unit
        rest, unit = (rest - term) * 16, unit / 16
        assert float(rest.abs().max()) <= 2.0 ** 15
    assert torch.equal(total, x.double())
