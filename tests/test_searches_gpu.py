"""Searches by beams and what runs beside them, on the device: orders that values do not tell, the front end on every kind of cache, adapters of several types."""
import numpy as np
import pytest
import torch

from conftest import load_pkg
from test_page_caches_gpu import begin, front_end, prompts_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def selected(ops, z, scores, k):
    scores, tokens, parents = ops.beam_select(torch.from_numpy(z).to(DEV), torch.tensor(scores, dtype=torch.float32, device=DEV), k=k)
    return scores.cpu(), tokens.cpu().tolist(), parents.cpu().tolist()


def test_logits_closer_than_their_values(ops):
    """Logits so small that their values are one number in 64 bits: a beam's order is still that of its logits, whatever columns they are in."""
    V = 5000
    z = np.zeros((1, V), np.float32)
    z[0, [4000, 10, 20, 4999, 700]] = 2e-20, 1e-20, 3e-20, 2e-20, -1e-20
    _, tokens, parents = selected(ops, z, [[-1.0]], 6)
    assert tokens == [[20, 4000, 4999, 10, 0, 1]] and parents == [[0] * 6]
    # descending columns, more of them than are asked for: the greatest, not the first
    z = np.zeros((1, V), np.float32)
    z[0, 100:140] = np.arange(1, 41, dtype=np.float32) * np.float32(2.0 ** -70)
    assert selected(ops, z, [[0.0]], 32)[1] == [list(range(139, 107, -1))]
    # between beams such values are equal, and the lower beam goes first
    z = np.zeros((3, V), np.float32)
    z[0, 77], z[1, 5], z[2, 9] = 1e-20, 9e-20, 5e-20
    _, tokens, parents = selected(ops, z, [[0.0, 0.0, 0.0]], 4)
    assert tokens == [[77, 0, 1, 2]] and parents == [[0, 0, 0, 0]]
    _, tokens, parents = selected(ops, z, [[-1.0, 0.0, -2.0]], 3)
    assert tokens == [[5, 0, 1]] and parents == [[1, 1, 1]]
