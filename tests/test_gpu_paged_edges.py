"""Attention of several sequences on a B200 at the edges of its contract: lengths that no table holds, scores that are all -inf, weights
far below the largest, wait limits, dependent launches. Helpers and the tolerance's derivation are test_gpu_paged's."""
import pytest

from test_gpu_paged import Pool, _check, _dt, _reference, _scratch, _starts

pytestmark = pytest.mark.gpu


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 257, 2 ** 30 + 1, -2 ** 31])
@pytest.mark.parametrize("new,max_new", [(1, 1), (3, 3), (3, None), (70, None)])
def test_a_length_that_cannot_be_leaves_the_others_alone(dev, length, new, max_new):
    """NaN (or, below zero, nothing seen) for the sequence that claims it; the others as they should be."""
    import torch
    lens = [300, 200, 129]
    pool = Pool(lens, 2, 128, 16, _dt("bf16"), 8)
    q = torch.randn(3 * new, 8, 128, device="cuda").bfloat16()
    out = torch.full((3 * new, 8, 128), 7.0, device="cuda")
    dev.AttnPaged(out, q, pool.kv, _starts([new] * 3), _i32([300, length, 129]), _scratch(dev), max_new=max_new, stream=_stream())
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    for s in (0, 2):
        ref, mag, size = _reference(q[s * new:(s + 1) * new], *pool.rows[s], lens[s] - new, 128 ** -0.5)
        _check(out[s * new:(s + 1) * new], ref, mag, size, _dt("bf16"), 300, 128)
    bad = out[new:2 * new]
    assert bool(bad.isnan().all()) if length > 0 else bool((bad == 0).all())
