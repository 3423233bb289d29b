"""The generator behind dropout: the numpy form that the GPU tests compare with against the method's published answers
(Salmon, Moraes, Dror and Shaw, 2011), of zeros, of ones and of the digits of pi, and the kernel at keys and places of
ones."""
import numpy as np
import pytest
import torch

import flow_b200 as fb
from test_gpu_dropout import bits, philox


@pytest.mark.parametrize("counter,key,want", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])])
def test_published_answers(counter, key, want):
    assert [int(w[0]) for w in philox([np.array([c], dtype=np.uint32) for c in counter], key)] == want


@pytest.mark.gpu
@pytest.mark.parametrize("key,place", [(-1, -1), (-1, 0), (0, -1), (-2 ** 63, 2 ** 63 - 1), (0xFFFFFFFF, -2 ** 32)])
def test_keys_and_places_of_ones(key, place):
    """The mask bit for bit, at thresholds about the first row's own bits, on rows of whole eights and of others."""
    ctx = fb.Context((0,))
    rng = torch.tensor([key, place], device="cuda")
    for rows, d in ((33, 264), (9, 77)):
        b = bits(rng, rows, d)
        x, y = torch.ones(rows, d, device="cuda"), torch.empty(rows, d, device="cuda")
        for cut in sorted({int(v) + e for v in b[0, :8] for e in (0, 1)} | {1, 65535}):
            ctx.dropout(fb.dropout_site(rows, d, torch.float32, cut / 65536), x, None, y, rng)
            assert ((y > 0).cpu().numpy() == (b >= cut)).all()
    ctx.close()
