"""GPU: ``policy.lm_head_token_logps`` at sizes chosen by the rule that picks its row tiles: every width, with and without
entropies, products kept and formed again, several tiles per workgroup and rows that do not fill the last one.

The tolerances are those of the module whose check this is (test_gpu_policy_head)."""

import pytest
import torch

from genrec_amd import _lib
from test_gpu_policy_head import _check, _inputs

def _row_tile(N, V, cus=256):
    """The rule, restated: least cost of whole rounds over the CUs, the wider tile where two cost the same."""
    cost = {64: 0.4, 128: 0.64, 192: 0.84, 256: 1.0}
    columns = (V + 255) // 256

    def rounds(bn):
        per_cu = 2 if bn == 64 else 1
        tiles = columns * ((N + bn - 1) // bn)
        return -(-tiles // (per_cu * cus)) * cost[bn] * per_cu

    return min(cost, key=lambda bn: (rounds(bn), -bn))


def _scratch(N, H, V, bn):
    """What the forward pass asks for with row tiles of bn (rows below 2^14)."""
    up = lambda n: (n + 255) // 256 * 256
    waves = {64: 8, 128: 4, 192: 4, 256: 2}[bn]  # parts that a tile of 256 columns leaves per row
    partials = (V + 255) // 256 * waves * ((N + bn - 1) // bn * bn) * 8
    return 256 + 3 * up(4 * N) + up(2 * N * H) + up(partials)


# (rows, H, V, tile): 593 tiles of columns at the real vocabulary, more than run at a time
CASES = [(5, 128, 151669, 64), (100, 128, 151669, 128), (320, 128, 151669, 192), (400, 64, 151669, 256), (400, 576, 151669, 256),
         (1400, 128, 151669, 256), (333, 192, 70001, 192), (2000, 64, 20000, 256)]


@pytest.mark.parametrize("N,H,V,tile", CASES)
def test_the_rule_picks_this_tile(N, H, V, tile):
    assert _row_tile(N, V) == tile
    assert _lib.lib().grx_lm_token_logps_scratch_bytes(N, H, V, 0) == _scratch(N, H, V, tile)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,V,tile", CASES)
def test_every_tile_with_and_without_entropies(N, H, V, tile):
    hidden, weight, ids, g, h = _inputs((N,), H, V, seed=N + H)
    _check(hidden, weight, ids, g, h, 0.8)  # kept and formed again
    _check(hidden, weight, ids, g, None, 1.0)
