"""The decoder's host logic without a GPU: positions of packed prompts and their rotation."""
import pytest
import torch

from jitllm_b200 import decoder


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("starts,n", [([0, 100], 512), ([0, 3, 3, 10], 10), ([0, 5, 5], 9), ([0, 0], 4), ([0, 700, 701], 701)])
def test_positions_of_packed_rows(starts, n):
    """Each row's position in its prompt; rows behind the last prompt sit at a position that any table has."""
    want = [0] * n
    for a, b in zip(starts, starts[1:]):
        want[a:b] = range(b - a)
    assert decoder.packed_positions(_i32(starts), n).tolist() == want


@pytest.mark.parametrize("starts,n,want", [([0, 3, 3, 10], 12, [2, 2, 9]), ([0, 0, 5], 5, [0, 4]), ([0, 4, 900], 8, [3, 7]), ([0, -7, 8], 8, [0, 7])])
def test_last_rows_are_rows(starts, n, want):
    """Starts that pass the rows or fall below zero index none outside them."""
    assert decoder.last_rows(_i32(starts), n).tolist() == want


def test_starts_without_a_prompt_are_refused():
    with pytest.raises(ValueError):
        decoder.packed_positions(_i32([0]), 4)


def test_rotation_is_that_of_the_tables_and_goes_on_behind_them():
    dec = decoder.Decoder.__new__(decoder.Decoder)
    dec.inv_freq = 1.0 / (10000.0 ** (torch.arange(0, 16, 2).float() / 16))
    cos, sin = dec._rotation(torch.arange(64))
    pos = torch.tensor([0, 63, 7, 500, 63])
    c, s = dec._rotation(pos)
    for i, p in enumerate(pos.tolist()):
        if p < 64:
            assert torch.equal(c[i], cos[p]) and torch.equal(s[i], sin[p])
    ang = 500.0 * dec.inv_freq.double()
    assert float((c[3] - ang.cos()).abs().max()) < 500 * 2.0 ** -23 and float((s[3] - ang.sin()).abs().max()) < 500 * 2.0 ** -23


@pytest.mark.parametrize("n", [0, 65, 4000])
def test_a_prompt_that_does_not_fit_the_caches_is_refused(n):
    """On the host, before the positions index a table."""
    dec = decoder.Decoder.__new__(decoder.Decoder)
    dec.torch, dec.max_len = torch, 64
    with pytest.raises(ValueError, match="max_len"):
        dec.prefill(torch.zeros(n, dtype=torch.int64))
