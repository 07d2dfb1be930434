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


@pytest.mark.parametrize("out", ["f32", "f16"])
@pytest.mark.parametrize("hq,hkv,d,new,n,exponent", [(8, 2, 128, 1, 131072, 18.1), (8, 8, 64, [1] * 70, 2500, 17.4), (8, 1, 64, 2, 70001, 17.4), (4, 2, 128, 40, 60000, 17.4),
                                                     (8, 4, 64, 300, 40000, 17.4), (16, 1, 128, 1, 5000, 15.3), (8, 2, 64, 33, 3000, 15.3)])
def test_a_long_flat_tail_keeps_its_weight(dev, out, hq, hkv, d, new, n, exponent):
    """f16, one position far above all others (by e^exponent, 2^22 to 2^26): together the others weigh up to a part in 500, each of them
    less than half of f16's smallest step beside one. The large position's value is zero, so that the tail is the result.
    A weight is held to 2^-39 of the largest, or to 2^-31 where many rows have 16-bit results: n times that of the largest value beside
    the tolerance of the other tests (without its allowance of n 2^-25 for this)."""
    import torch
    from jitllm_b200 import PagedKV
    each = new if isinstance(new, list) else [new]                          # one sequence whose parts are joined, or many whole ones
    new = sum(each)
    pool = Pool([n], hkv, d, 64, torch.float16, 5)
    k, v = pool.rows[0]
    k.zero_()
    k[3, :, 0] = 1.0
    v.abs_().add_(0.25)
    v[3] = 0
    p = torch.arange(n, device="cuda")
    page = pool.table[0].long()[p // 64]
    pool.k[page, :, p % 64], pool.v[page, :, p % 64] = k, v
    kv = PagedKV(pool.k, pool.v, pool.table.expand(len(each), -1).contiguous())
    q = torch.randn(new, hq, d, device="cuda").half()
    q[..., 0] = exponent
    res = torch.full((new, hq, d), 7.0, device="cuda", dtype=_dt(out))
    dev.AttnPaged(res, q, kv, _starts(each), _i32([n] * len(each)), _scratch(dev), max_new=max(each), scale=1.0, stream=_stream())
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    if len(each) > 1:
        ref, mag, size = (torch.cat(x) for x in zip(*(_reference(q[i:i + 1], k, v, n - 1, 1.0) for i in range(new))))
    else:
        ref, mag, size = _reference(q, k, v, n - new, 1.0)
    few = max(each) * hq // hkv <= 16
    w = 2.0 ** -22 if few or out == "f32" else 2.0 ** -11
    floor = 2.0 ** -39 if few or out == "f32" else 2.0 ** -31
    e = size * (d * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -22
    tol = mag * (w + 2 * e + (128 + n / 128) * 2.0 ** -23) + n * floor * float(v.max())
    h = torch.finfo(_dt(out))
    tol = tol + ref.abs() * h.eps / 2 + h.smallest_normal * h.eps / 2
    bad = (res.double() - ref).abs() > tol
    assert not bool(bad.any()), float(((res.double() - ref).abs() / tol).max())


def _exact_scores(rows, hq, hkv, d, n, dt, seed):
    """q, k, v whose scores, at a scale of log 2, are multiples of 1/32 up to 4 that no product or sum rounds."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def steps(k, *shape):
        return torch.randint(0, k + 1, shape, generator=g, device="cuda")
    q, k = torch.zeros(rows, hq, d, device="cuda", dtype=dt), torch.zeros(n, hkv, d, device="cuda", dtype=dt)
    q[..., 0] = (steps(16, rows, hq) / 8).to(dt)                           # up to 2, in eighths
    k[..., 0] = (steps(8, n, hkv) / 4).to(dt)                              # up to 2, in quarters
    v = torch.randn(n, hkv, d, generator=g, device="cuda").to(dt)
    return q, k, v


def _weights_of_24_bits(got, ref, mag, n):
    """f32 results of exact scores. Of A = sum p|v| / sum p: 2^-22 for a weight as 16-bit parts; its exponent, twice (in the sum and in the
    product): 2^-22 of the exponential, 4 * 2^-24 of the scale's two roundings at exponents up to 4, 2^-23 of their product's; n + 8 additions
    in f32 that may truncate, 2^-23 each; 3 * 2^-24 for the quotient."""
    tol = mag * (2.0 ** -22 + 2 * (2.0 ** -22 + 4 * 2.0 ** -24 + 2.0 ** -23) + (n + 8) * 2.0 ** -23 + 3 * 2.0 ** -24) + 1e-30
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), float(((got.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (12, 4, 64), (16, 1, 128)])
def test_f32_results_of_few_rows_carry_f32_weights(dev, dt, hq, hkv, d):
    """A weight in two bf16 values would be off by up to 2^-16."""
    import torch
    from jitllm_b200 import PagedKV
    lens, scale = [8, 7, 5, 2, 1, 8, 6, 3] * 8, float(torch.tensor(2.0).log())
    q, k, v = _exact_scores(len(lens), hq, hkv, d, 8 * len(lens), _dt(dt), 3)
    pk, pv = (torch.zeros(len(lens), hkv, 16, d, device="cuda", dtype=_dt(dt)) for _ in range(2))
    pk[:, :, :8], pv[:, :, :8] = (x.view(len(lens), 8, hkv, d).transpose(1, 2) for x in (k, v))
    table = torch.arange(len(lens), device="cuda", dtype=torch.int32)[:, None].contiguous()
    out = torch.empty(len(lens), hq, d, device="cuda")
    dev.AttnPaged(out, q, PagedKV(pk, pv, table), _starts([1] * len(lens)), _i32(lens), _scratch(dev), max_new=1, scale=scale, stream=_stream())
    torch.cuda.synchronize()
    for s, n in enumerate(lens):
        ref, mag, _ = _reference(q[s:s + 1], k[8 * s:8 * s + n], v[8 * s:8 * s + n], n - 1, scale)
        _weights_of_24_bits(out[s:s + 1], ref, mag, n)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,nseq", [(8, 8, 128, 40), (12, 4, 64, 9), (16, 1, 128, 30), (16, 1, 64, 1)])
def test_f32_results_of_many_rows_carry_f32_weights(dev, dt, hq, hkv, d, nseq):
    """Prompts of up to eight tokens, packed: the tensor core's kernel with one tile and with two."""
    import torch
    new = [8, 7, 5, 2, 1, 8, 6, 3][:nseq] * (nseq // 8) + [8] * (nseq % 8)
    scale = float(torch.tensor(2.0).log())
    q, k, v = _exact_scores(sum(new), hq, hkv, d, sum(new), _dt(dt), 4)
    out = torch.empty(sum(new), hq, d, device="cuda")
    dev.AttnPrompt(out, q, k, v, _starts(new), _scratch(dev), scale=scale, stream=_stream())
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    at = 0
    for n in new:
        ref, mag, _ = _reference(q[at:at + n], k[at:at + n], v[at:at + n], 0, scale)
        _weights_of_24_bits(out[at:at + n], ref, mag, 8)
        at += n


def _programmatic_edges(graph):
    """Of a captured graph's edges, those along which a kernel may start before the one in front of it is done."""
    import ctypes as C
    cu = C.CDLL("libcuda.so.1")
    h, n = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert cu.cuGraphGetEdges_v2(h, None, None, None, C.byref(n)) == 0
    a, b, data = (C.c_void_p * n.value)(), (C.c_void_p * n.value)(), (C.c_uint8 * (8 * n.value))()      # from, to; ports, type, reserved
    assert cu.cuGraphGetEdges_v2(h, a, b, data, C.byref(n)) == 0
    return sum(data[8 * i + 2] == 1 for i in range(n.value))


def test_no_dependent_launches_where_the_context_forbids_them():
    import torch
    from jitllm_b200 import Device, PagedKV, _lib
    cos, q = torch.zeros(64, 32, device="cuda"), torch.zeros(40, 8, 64, device="cuda", dtype=torch.bfloat16)
    qkv, lens, table = torch.randn(40, 12 * 64, device="cuda"), _i32([40, 50]), torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
    kv = PagedKV(torch.zeros(8, 2, 128, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(8, 2, 128, 64, device="cuda", dtype=torch.bfloat16), table)
    found, results = [], []
    for flags in (0, _lib.FLAG_NO_PDL):
        with Device(0, flags=flags) as d:
            out, starts, scratch = torch.zeros(40, 8, 64, device="cuda"), _starts([1, 39]), _scratch(d)

            def calls(stream):
                d.RopeAppend(q, qkv, kv, starts, lens, cos + 1, cos, stream=stream)
                d.AttnPaged(out, q, kv, starts, lens, scratch, max_new=39, stream=stream)        # few rows, many rows, a join of each
                d.AttnPrompt(out, q, q[:, :2], q[:, 2:4], starts, scratch, stream=stream)
            calls(_stream())
            torch.cuda.synchronize()
            results.append(out.clone())
            graph = torch.cuda.CUDAGraph(keep_graph=True)
            with torch.cuda.graph(graph):
                calls(_stream())
            found.append(_programmatic_edges(graph))
            graph.reset()
    assert found[0] >= 5 and found[1] == 0 and torch.equal(*results)


def _last_of_a_million(d, rows):
    """A prompt behind 2^20 - 1 sequences without rows: each CTA goes over all of them before it knows its share. (out, check)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(rows, h, 128, generator=g, device="cuda").bfloat16() for h in (8, 2, 2))
    starts = torch.zeros((1 << 20) + 1, dtype=torch.int32, device="cuda")
    starts[-1] = rows
    out = torch.full((rows, 8, 128), 7.0, device="cuda")
    d.AttnPrompt(out, q, k, v, starts, _scratch(d), stream=_stream())
    torch.cuda.synchronize()
    return out, lambda o: _check(o, *_reference(q, k, v, 0, 128 ** -0.5), _dt("bf16"), rows, 128)


def test_a_wait_that_runs_out_is_reported_and_the_context_goes_on():
    """With a limit of a microsecond the roles that wait for a share give up (after 4 ms: they are patient) before a walk over a million
    sequences has found one: the kernel returns, the status says so, and the next call is right."""
    import torch
    from jitllm_b200 import Device
    with Device(0, wait_limit_us=1) as d:
        _last_of_a_million(d, 300)
        assert not d.StatusPoll() and "attention" in d.Err()
        assert d.StatusPoll()
        q = torch.randn(4, 8, 128, device="cuda").bfloat16()                # sixteen query rows: a kernel that waits for nothing
        out = torch.empty_like(q)
        d.AttnPrompt(out, q, q[:, :2], q[:, 2:4], _starts([4]), _scratch(d), stream=_stream())
        torch.cuda.synchronize()
        _check(out, *_reference(q, q[:, :2], q[:, 2:4], 0, 128 ** -0.5), _dt("bf16"), 4, 128)
        assert d.StatusPoll()
    with Device(0) as d:
        out, check = _last_of_a_million(d, 300)
        assert d.StatusPoll()
        check(out)


@pytest.mark.parametrize("new,lens", [([20] * 200, [9000] * 200), ([60] * 100, [9000] * 100)])
def test_a_short_limit_does_not_end_long_work(new, lens):
    """Two tiles to an item, the second one idle: its roles wait through all of the first one's work, many times the limit."""
    import torch
    from jitllm_b200 import Device, PagedKV
    g = torch.Generator(device="cuda").manual_seed(6)
    pages = torch.randn(160, 2, 64, 128, generator=g, device="cuda").bfloat16()
    table = torch.stack([torch.randperm(160, generator=g, device="cuda")[:lens[0] // 64 + 1] for _ in new]).to(torch.int32)
    q = torch.randn(sum(new), 2, 128, generator=g, device="cuda").bfloat16()
    kv, st = PagedKV(pages, pages.flip(0).contiguous(), table), _stream()
    got = []
    for limit in (0, 60):
        with Device(0, wait_limit_us=limit) as d:
            out = torch.zeros_like(q)
            d.AttnPaged(out, q, kv, _starts(new), _i32(lens), _scratch(d), stream=st)
            torch.cuda.synchronize()
            assert d.StatusPoll()
            got.append(out)
    assert torch.equal(*got)


@pytest.mark.parametrize("rows", [3, 12, 200])
@pytest.mark.parametrize("what", ["kv heads", "kv rows", "q heads", "q rows", "overlapping rows", "far rows"])
def test_strides_that_repeat_overlap_or_leap(dev, rows, what):
    """Views whose strides are zero, smaller than a row or large: on the kernel for few rows and on the tensor core's."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(12)
    hq, hkv, d = 8, 4, 64

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()
    q, k, v = randn(rows, hq, d), randn(rows, hkv, d), randn(rows, hkv, d)
    if what == "kv heads":
        k, v = k[:, :1].expand(-1, hkv, -1), v[:, :1].expand(-1, hkv, -1)
    elif what == "kv rows":
        k, v = k[:1].expand(rows, -1, -1), v[:1].expand(rows, -1, -1)
    elif what == "q heads":
        q = q[:, :1].expand(-1, hq, -1)
    elif what == "q rows":
        q = q[:1].expand(rows, -1, -1)
    elif what == "overlapping rows":
        q, k, v = (randn(8 * rows + h * d).as_strided((rows, h, d), (8, d, 1)) for h in (hq, hkv, hkv))
    else:
        q, k, v = (randn(h * 8192 + rows * d).as_strided((rows, h, d), (d, 8192, 1)) if rows * d <= 8192 else
                   randn(rows * 8192).as_strided((rows, h, d), (8192, d, 1)) for h in (hq, hkv, hkv))
    for dt in ("f32", "bf16"):
        out = torch.full((rows, hq, d), 7.0, device="cuda", dtype=_dt(dt))
        dev.AttnPrompt(out, q, k, v, _starts([rows]), _scratch(dev), stream=_stream())
        torch.cuda.synchronize()
        assert dev.StatusPoll()
        _check(out, *_reference(q, k, v, 0, d ** -0.5), torch.bfloat16, rows, d)


@pytest.mark.parametrize("hq,hkv,d", [(1024, 64, 64), (300, 300, 128), (1000, 125, 64)])
@pytest.mark.parametrize("new,max_new", [([1, 0, 2], 2), ([1, 70, 20], None)])
def test_hundreds_of_heads(dev, hq, hkv, d, new, max_new):
    import torch
    lens = [33, 80, 150]
    pool = Pool(lens, hkv, d, 16, _dt("bf16"), 2)
    q = torch.randn(sum(new), hq, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    out = torch.full((sum(new), hq, d), 7.0, device="cuda", dtype=torch.bfloat16)
    dev.AttnPaged(out, q, pool.kv, _starts(new), _i32(lens), _scratch(dev), max_new=max_new, stream=_stream())
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    at = 0
    for s, n in enumerate(new):
        _check(out[at:at + n], *_reference(q[at:at + n], *pool.rows[s], lens[s] - n, d ** -0.5), _dt("bf16"), lens[s], d)
        at += n


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", [(3, 2, 4), (5, 1, 12), (2, 2, 96), (4, 1, 256), (2, 1, 1024), (1, 600, 8)])
def test_the_writer_takes_any_multiple_of_four(dev, x, hq, hkv, d):
    """Head sizes that the attention does not serve. One rounding to the cache's type of a result that is off by 2^-24 for each of two
    products and their sum."""
    import torch
    from jitllm_b200 import PagedKV
    new, lens, p = [3, 1, 20], [3, 17, 45], 16
    table = torch.arange(9, device="cuda", dtype=torch.int32).flip(0).view(3, 3)
    k = torch.full((9, hkv, p, d), 7.0, device="cuda", dtype=torch.bfloat16)
    v = torch.full_like(k, 7.0)
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(25, (hq + 2 * hkv) * d, device="cuda", generator=g).to(_dt(x))
    ang = torch.arange(64, device="cuda")[:, None] * 0.7 ** torch.arange(d // 2, device="cuda")[None, :]
    cos, sin = ang.cos(), ang.sin()
    q = torch.full((25, hq, d), 7.0, device="cuda", dtype=torch.bfloat16)
    dev.RopeAppend(q, qkv, PagedKV(k, v, table), _starts(new), _i32(lens), cos, sin, stream=_stream())
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
    seq = torch.cat([torch.full((m,), s, device="cuda") for s, m in enumerate(new)])
    rows = qkv[:24].double().view(24, hq + 2 * hkv, d)
    a, b = rows[:, :hq + hkv, 0::2], rows[:, :hq + hkv, 1::2]
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    rot, size = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), (a.abs() + b.abs()).repeat_interleave(2, -1)
    page, slot = table[seq, pos // p].long(), pos % p
    tol = rot.abs() * 2.0 ** -8 + size * 3 * 2.0 ** -24 * (1 + 2.0 ** -8)
    assert not bool(((q[:24].double() - rot[:, :hq]).abs() > tol[:, :hq]).any()) and bool((q[24] == 7.0).all())
    assert not bool(((k[page, :, slot].double() - rot[:, hq:]).abs() > tol[:, hq:]).any())
    assert torch.equal(v[page, :, slot], rows[:, hq + hkv:].to(torch.bfloat16))
    k[page, :, slot], v[page, :, slot] = 7.0, 7.0
    assert bool((k == 7.0).all()) and bool((v == 7.0).all())               # nothing else was written


@pytest.mark.parametrize("scale", [3.0e38, float("inf"), float("nan"), 0.0, -1.0])
def test_a_scale_that_leaves_f32_is_refused(dev, scale):
    """To the base 2 a scale is 1.44 times as large: past 2.35e38 it would be infinite, and a score of zero not a number."""
    import torch
    from jitllm_b200 import DeviceError, _lib
    q = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(DeviceError) as e:
        dev.AttnPrompt(torch.empty_like(q), q, q, q, _starts([4]), _scratch(dev), scale=scale)
    assert e.value.status == _lib.EINVAL
