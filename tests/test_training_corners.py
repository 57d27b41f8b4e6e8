"""Corners of the training operators that need no GPU."""
import torch

from mvs_amd import synth
from mvs_amd.models import matching_cells


def test_matching_cells_of_a_map_beyond_2_to_24_cells():
    """A cell's number is a whole number throughout: float32 has every second one only from 2^24 on."""
    h, w = 4099, 4097
    proj = torch.from_numpy(synth.proj_matrices(2, h, w)).expand(1, -1, -1, -1)
    cells = matching_cells(torch.full((1, h, w), 600.0), proj[:, 0], proj[:, 0])[0]
    want = torch.arange(h * w)
    assert torch.equal(cells[cells >= 0], want[cells >= 0]) and int((cells < 0).sum()) <= 2 * (h + w)
