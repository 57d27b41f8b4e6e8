"""Corners of the training operators that need no GPU."""
import pytest
import torch

from mvs_amd import synth
from mvs_amd.models import matching_cells
from product_pieces import LOW_PIECES, PAIRS, SCALE, gradient_bound, gradient_case, gradient_errors, logit_case, product_of


def test_matching_cells_of_a_map_beyond_2_to_24_cells():
    """A cell's number is a whole number throughout: float32 has every second one only from 2^24 on."""
    h, w = 4099, 4097
    proj = torch.from_numpy(synth.proj_matrices(2, h, w)).expand(1, -1, -1, -1)
    cells = matching_cells(torch.full((1, h, w), 600.0), proj[:, 0], proj[:, 0])[0]
    want = torch.arange(h * w)
    assert torch.equal(cells[cells >= 0], want[cells >= 0]) and int((cells < 0).sum()) <= 2 * (h + w)


# ------------------------------------------------------------------ the cases of the low pieces see what they are made to see
def _logit_error(which, product, n, V, C):
    x, w, want = logit_case(which, n, V, C)
    return float((SCALE * (product(x, w).double() - want.double())).abs().max())


def _gradient_error(product, n, V, C):
    x, w, of_x, of_w = gradient_case(n, V, C)
    t = torch.full((n,), V - 1)
    dl = torch.full((n, V), 1.0 / V)
    dl[:, V - 1] -= 1
    gx, gw = product(dl, w.t().contiguous()), product(dl.t().contiguous(), x.t().contiguous())
    return gradient_errors(V, gx, gw, t, of_x, of_w)


@pytest.mark.parametrize("n,V,C", LOW_PIECES)
def test_a_product_without_one_of_the_low_pieces_would_be_seen(n, V, C):
    for which in PAIRS[:3]:
        assert _logit_error(which, product_of(PAIRS), n, V, C) == 0
        without = product_of([p for p in PAIRS if p != which])
        assert _logit_error(which, without, n, V, C) > 1
        assert _gradient_error(without, n, V, C) > 2 * gradient_bound(V), which
    assert _gradient_error(product_of(PAIRS), n, V, C) <= gradient_bound(V)
    assert _gradient_error(lambda a, b: a @ b.t(), n, V, C) <= gradient_bound(V)
