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


@pytest.mark.parametrize("dt,d", [("bf16", 128), ("f16", 128), ("bf16", 64), ("f16", 64)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("new,max_new", [(1, 1), (4, 4), (20, 20), (90, None)])
def test_scores_that_are_all_minus_infinity_have_no_result(dev, dt, d, out, new, max_new):
    """0 / 0 by the definition: NaN, whether an item is whole or in parts. Where some positions' scores are finite, the others weigh nothing."""
    import torch
    lens, dark = [100, 150, 9000, 9000, 0], [100, 60, 9000, 7000, 0]       # the first `dark` keys of each are infinite
    if new > 60:
        lens[0], dark[0] = 120, 120
    pool = Pool(lens, 2, d, 32, _dt(dt), 4)
    g = torch.Generator(device="cuda").manual_seed(9)
    for s, n in enumerate(dark):
        p = torch.arange(n, device="cuda")
        pool.k[pool.table[s].long()[p // 32], :, p % 32, 5] = float("inf")
    q = torch.randn(5 * new, 8, d, generator=g, device="cuda").to(_dt(dt))
    q[..., 5] = -1.5
    res = torch.full((5 * new, 8, d), 7.0, device="cuda", dtype=_dt(out))
    dev.AttnPaged(res, q, pool.kv, _starts([new] * 5), _i32(lens), _scratch(dev), max_new=max_new, stream=_stream())
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    for s, (n, m) in enumerate(zip(lens, dark)):
        got, rows = res[s * new:(s + 1) * new], q[s * new:(s + 1) * new]
        if n == 0:
            assert bool((got == 0).all())                                  # these see nothing
        elif m == n:
            assert bool(got.isnan().all())
        else:
            k, v = (x[m:] for x in pool.rows[s])
            ref, mag, size = _reference(rows, k, v, n - m - new, d ** -0.5)
            first = max(0, m + new - n)                                    # rows that see infinite keys alone
            assert first == 0 or bool(got[:first].isnan().all())
            _check(got[first:], ref[first:], mag[first:], size[first:], _dt(dt), n, d)
