"""Few rows of wide 4-bit weights, as a vocabulary's: codes are taken as they are, wherever their rows lie."""

import pytest
import torch

import linear_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fo():
    import feather_ops

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return feather_ops


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [33, 50, 64])
def test_few_rows_of_wide_weights_are_not_rounded(fo, m, gated, aligned):
    """In float16 a weight of 15 times a scale of 5000 rounds to infinity."""
    n, k, group = 151940, 2048, 128
    g = torch.Generator("cuda").manual_seed(m)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    if not aligned:   # rows on 4-byte boundaries
        wide = torch.zeros((n, k // 2 + 4), device="cuda", dtype=torch.uint8)
        wide[:, 4:] = codes
        codes = wide[:, 4:]
    scale = torch.full((k // group, n), 5000.0, device="cuda").half().t()
    zero = torch.zeros((k // group, n), device="cuda", dtype=torch.uint8).t()
    x = (torch.randn((m, k), generator=g, device="cuda") * 1e-4).half()
    rows = torch.tensor([0, 1, 70000, n // 2 - 1, n // 2, n // 2 + 7, n - 2, n - 1], device="cuda")
    want, bound = ref.int4(x, codes[rows], scale[rows], zero[rows], None)
    assert ref.int4_values(codes[rows], scale[rows], zero[rows], k).half().isinf().any()
    if not gated:
        y = fo.int4_linear(x, codes, scale, zero)
        assert y.isfinite().all()
        ref.check(y[:, rows], want, bound)
        return
    y = fo.int4_gated_linear(x, codes, scale, zero)
    pairs = torch.tensor([0, 1, 70000, n // 2 - 1], device="cuda")
    both, off = ref.int4(x, codes[torch.cat((pairs, n // 2 + pairs))], scale[torch.cat((pairs, n // 2 + pairs))],
                         zero[torch.cat((pairs, n // 2 + pairs))], None)
    (gate, up), (d_gate, d_up) = both.chunk(2, 1), off.chunk(2, 1)
    value, slope = ref.activation(gate, "silu")
    off = (slope.abs() + 2 * d_gate) * d_gate * up.abs() + value.abs() * d_up + d_gate * d_up + ref.ACT * (value * up).abs()
    finite = (value * up).abs() < 60000   # a product of two large sums may be past the type
    assert finite.any() and y[:, pairs][finite].isfinite().all()
    off = (y[:, pairs].double() - value * up).abs() - off - ref.half_step(torch.float16, (value * up).abs() + off)
    assert (off[finite] <= 0).all()
