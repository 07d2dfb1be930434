"""Several sequences at once on a B200, against float64: attention over packed prompts (AttnPrompt), attention of new rows over a cache
in pages (AttnPaged), the cache's writer (RopeAppend), and the three together.

Tolerances. With A = sum p|v| / sum p of an output value (at least its magnitude), the result may differ from the exact one by
  A * (w + 2 e)   and   half a step of the output's type relative to the value,
where w is the rounding of the softmax weights -- half a step of the 16-bit type (bf16 2^-8, f16 2^-11), or for f32 results its square,
since two 16-bit values carry a weight -- and e the error of a weight's exponent: d additions of the score in f32, each off by at most
2^-23 of the terms' magnitude, the scaled exponent's own rounding, and 2^-22 of the exponential. Sums of n weights in f32 are within
n 2^-24 of A in the worst order; the tensor cores add at most 128 positions at a time and the running sums are as many as there are
such groups, so (128 + n / 128) 2^-23 stands for them. f16 weights below 2^-14 of the largest are held to 2^-25 of it at best: n 2^-25."""
import pytest

pytestmark = pytest.mark.gpu


def _half_step(dt):
    import torch
    return torch.finfo(dt).eps / 2


def _reference(q, k, v, pos0, scale):
    """q [n][hq][d], k, v [len][hkv][d] (16 bits): float64 results and the A and exponent magnitudes of the tolerance."""
    import torch
    n, hq, d = q.shape
    ln, hkv = k.shape[0], k.shape[1]
    g = hq // hkv
    out = torch.zeros(n, hq, d, device=q.device, dtype=torch.float64)
    mag = torch.zeros_like(out)
    size = torch.zeros(n, hq, 1, device=q.device, dtype=torch.float64)
    for i0 in range(0, n, 256):
        for h in range(hq):
            qq = q[i0:i0 + 256, h].double()
            see = torch.arange(i0, i0 + qq.shape[0], device=q.device)[:, None] + pos0 >= torch.arange(ln, device=q.device)[None, :]
            live = see.any(1)
            if ln == 0 or not bool(live.any()):
                continue
            kk, vv = k[:, h // g].double(), v[:, h // g].double()
            s = torch.where(see, qq @ kk.T * scale, -float("inf"))
            a = torch.where(see, qq.abs() @ kk.abs().T * scale, 0.0)
            p = torch.where(live[:, None], torch.softmax(s, -1), 0.0)
            vv0 = torch.where(see.any(0)[:, None], vv, 0.0)
            r = slice(i0, i0 + qq.shape[0])
            out[r, h], mag[r, h], size[r, h, 0] = p @ vv0, p @ vv0.abs(), a.amax(-1)
    return out, mag, size


def _check(got, ref, mag, size, in_dt, n_pos, d):
    import torch
    w = _half_step(in_dt)
    if got.dtype == torch.float32:
        w = w * w
    e = size * (d * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -22
    tol = mag * (w + 2 * e + (128 + n_pos / 128) * 2.0 ** -23)
    if in_dt == torch.float16:
        tol = tol + mag * n_pos * 2.0 ** -25
    tol = tol + ref.abs() * _half_step(got.dtype) + torch.finfo(got.dtype).smallest_normal
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - ref).abs() / tol).nan_to_num(1e9).max()))


def _starts(new, shift=0):
    import torch
    at = [shift]
    for n in new:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _scratch(dev):
    import torch
    return torch.randint(0, 256, (dev.AttnScratchBytes(),), device="cuda", dtype=torch.uint8)      # any state


class Pool:
    """A cache in pages, filled for sequences of the given lengths; every place that no sequence owns is NaN."""

    def __init__(self, lens, hkv, d, page_len, dt, seed, extra=3, spare=1):
        import torch
        from jitllm_b200 import PagedKV
        g = torch.Generator(device="cuda").manual_seed(seed)
        pages = [-(-n // page_len) for n in lens]
        total = sum(pages) + extra
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(pages + [0]) + spare), -1, dtype=torch.int32, device="cuda")
        self.k = torch.full((total, hkv, page_len, d), float("nan"), device="cuda", dtype=dt)
        self.v = torch.full_like(self.k, float("nan"))
        self.rows, at = [], 0
        for s, n in enumerate(lens):
            own = order[at:at + pages[s]]
            at += pages[s]
            self.table[s, :pages[s]] = own
            k, v = (torch.randn(n, hkv, d, generator=g, device="cuda").to(dt) for _ in range(2))
            where = torch.arange(n, device="cuda")
            page = own.long()[where // page_len] if n else where
            self.k[page, :, where % page_len], self.v[page, :, where % page_len] = k, v
            self.rows.append((k, v))
        self.kv = PagedKV(self.k, self.v, self.table)


def _paged_case(dev, new, lens, hq, hkv, d, page_len, dt, out_dt, seed, max_new=None, pad=2, scale=None, sharp=1.0):
    import torch
    pool = Pool(lens, hkv, d, page_len, dt, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    total = sum(new) + pad
    q = (torch.randn(total, hq, d, generator=g, device="cuda") * sharp).to(dt)
    out = torch.full((total, hq, d), 7.0, device="cuda", dtype=out_dt)
    starts, ln = _starts(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    dev.AttnPaged(out, q, pool.kv, starts, ln, _scratch(dev), max_new=max_new, scale=scale,
                  stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    assert bool((out[sum(new):] == 7.0).all())                          # rows behind the last sequence
    at = 0
    for s, n in enumerate(new):
        ref, mag, size = _reference(q[at:at + n], *pool.rows[s], lens[s] - n, d ** -0.5 if scale is None else scale)
        _check(out[at:at + n], ref, mag, size, dt, lens[s], d)
        at += n
    return out


DTS = ["bf16", "f16"]


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hq,hkv,d,page_len", [(32, 8, 128, 16), (8, 8, 64, 32), (4, 1, 128, 64), (9, 3, 64, 16), (10, 2, 128, 128), (16, 1, 64, 1024),
                                               (7, 1, 128, 256)])
def test_paged_single_tokens(dev, dt, hq, hkv, d, page_len):
    """One new token to a sequence: lengths of one, around tiles and pages, long ones; an idle and an empty sequence among them."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 1000, 2049, 40]
    new = [1] * 12 + [0, 1, 1, 0]
    _paged_case(dev, new, lens, hq, hkv, d, page_len, _dt(dt), _dt("f32"), 11 + hq, max_new=1)
    _paged_case(dev, new, lens, hq, hkv, d, page_len, _dt(dt), _dt(dt), 12 + hq, max_new=1, sharp=3.0)


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,lens", [(32, 8, 128, [20001]), (16, 2, 128, [70000]), (2, 2, 64, [9000, 1, 33000])])
def test_paged_long_sequences_are_divided(dev, out, hq, hkv, d, lens):
    a = _paged_case(dev, [1] * len(lens), lens, hq, hkv, d, 32, _dt("bf16"), _dt(out), 5, max_new=1)
    b = _paged_case(dev, [1] * len(lens), lens, hq, hkv, d, 32, _dt("bf16"), _dt(out), 5, max_new=1)
    assert bool((a == b).all())                                         # the same bits every time


@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("hq,hkv,d,page_len", [(32, 8, 128, 16), (8, 8, 64, 64), (9, 3, 128, 32), (10, 2, 64, 256), (16, 1, 128, 16)])
def test_paged_chunks(dev, dt, out, hq, hkv, d, page_len):
    """Several new rows to a sequence, over what is cached already and over nothing; idle sequences and single tokens among them."""
    new = [5, 0, 130, 1, 33, 64, 0, 257, 2]
    lens = [5, 400, 130, 77, 500, 64, 0, 1000, 129]
    _paged_case(dev, new, lens, hq, hkv, d, page_len, _dt(dt), _dt(out), 3 + d)
    _paged_case(dev, new[:6], lens[:6], hq, hkv, d, page_len, _dt(dt), _dt(out), 4 + d, max_new=130, scale=0.31)


@pytest.mark.parametrize("max_new", [1, 3, 16, None])
def test_the_hint_picks_the_kernel_not_the_result(dev, max_new):
    _paged_case(dev, [3, 40, 1], [90, 40, 2000], 8, 2, 128, 16, _dt("bf16"), _dt("bf16"), 21, max_new=max_new)


def test_sequences_shorter_than_their_new_rows(dev):
    """Rows before position 0 see nothing: zeros."""
    import torch
    for max_new in (1, None):
        pool = Pool([2, 100, 0], 2, 128, 16, _dt("bf16"), 1)
        q = torch.randn(140, 8, 128, device="cuda").bfloat16()
        out = torch.full((140, 8, 128), 7.0, device="cuda")
        starts, lens = _starts([5, 105, 30]), torch.tensor([2, 100, 0], dtype=torch.int32, device="cuda")
        dev.AttnPaged(out, q, pool.kv, starts, lens, _scratch(dev), max_new=max_new, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert bool((out[:3] == 0).all()) and bool((out[5:10] == 0).all()) and bool((out[110:] == 0).all())
        for a, b, s in ((3, 5, 0), (10, 110, 1)):
            ref, mag, size = _reference(q[a:b], *pool.rows[s], 0, 128 ** -0.5)
            _check(out[a:b], ref, mag, size, _dt("bf16"), 100, 128)


@pytest.mark.parametrize("max_new", [1, None])
def test_bad_pages_are_not_followed(dev, max_new):
    """Page numbers outside the pool and lengths beyond the table: NaN for that sequence, the others as they should be."""
    import torch
    lens, new = [70, 90, 300, 64], [2, 2, 2, 1]
    pool = Pool(lens, 2, 128, 16, _dt("bf16"), 8)
    pool.table[0, 1] = -5
    pool.table[1, 3] = pool.k.shape[0]
    pool.table[2, 7] = 2 ** 31 - 1
    q = torch.randn(7, 8, 128, device="cuda").bfloat16()
    out = torch.zeros(7, 8, 128, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dev.AttnPaged(out, q, pool.kv, _starts(new), lens_d, _scratch(dev), max_new=max_new, stream=st)
    torch.cuda.synchronize()
    assert bool(out[:6].isnan().all())
    ref, mag, size = _reference(q[6:], *pool.rows[3], 63, 128 ** -0.5)
    _check(out[6:], ref, mag, size, _dt("bf16"), 64, 128)
    lens_d[3] = 16 * pool.table.shape[1] + 40                            # more than the table holds
    out.zero_()
    dev.AttnPaged(out, q, pool.kv, _starts(new), lens_d, _scratch(dev), max_new=max_new, stream=st)
    torch.cuda.synchronize()
    assert bool(out[6:].isnan().all())


@pytest.mark.parametrize("max_new", [4, 20, None])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(dev, max_new, value):
    """Infinite or NaN keys and values at a sequence's own later positions leave its earlier rows alone."""
    import torch
    lens, new = [75, 300], [4, 150]
    pool = Pool(lens, 2, 128, 16, _dt("bf16"), 8)
    for s, p in ((0, 73), (1, 200)):                                     # row 2 of 4; row 50 of 150
        page, slot = int(pool.table[s, p // 16]), p % 16
        pool.k[page, :, slot, 5] = value
        pool.v[page, 0, slot, 9] = value
        pool.v[page, 1, slot, 100] = -value
    q = torch.randn(154, 8, 128, device="cuda").bfloat16()
    out = torch.zeros(154, 8, 128, device="cuda", dtype=torch.bfloat16)
    dev.AttnPaged(out, q, pool.kv, _starts(new), torch.tensor(lens, dtype=torch.int32, device="cuda"), _scratch(dev), max_new=max_new,
                  stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for a, n, s in ((0, 2, 0), (4, 50, 1)):
        ref, mag, size = _reference(q[a:a + n], *pool.rows[s], lens[s] - new[s], 128 ** -0.5)
        _check(out[a:a + n], ref, mag, size, _dt("bf16"), 300, 128)
    assert not bool(out[54:].isfinite().all(-1).any())                   # the rows that see them do


@pytest.mark.parametrize("new", [1, 6, 40])
def test_many_sequences(dev, new):
    """More than a warp looks over at once, of all lengths, some idle or empty."""
    lens = [(37 * s * s) % 700 for s in range(300)]
    n = [0 if s % 7 == 3 else min(new, lens[s]) for s in range(300)]
    _paged_case(dev, n, lens, 8, 2, 64, 32, _dt("bf16"), _dt("bf16"), 9, max_new=new)


@pytest.mark.parametrize("hq,d,new,n", [(4, 128, 1, 70001), (8, 64, 2, 60000), (16, 64, 5, 20011), (16, 128, 20, 20011), (1, 64, 300, 40000)])
def test_one_item_in_hundreds_of_parts(dev, hq, d, new, n):
    """One kv head of one sequence: its few items are all the work, and each is divided over as many CTAs as there are."""
    _paged_case(dev, [new], [n], hq, 1, d, 256, _dt("bf16"), _dt("f32"), n + new)
    _paged_case(dev, [new, 1], [n, 900], hq, 1, d, 64, _dt("f16"), _dt("f16"), n)


@pytest.mark.parametrize("new,lens", [([1] * 9, [48, 1, 33, 2, 16, 17, 47, 5, 40]), ([1] * 300, [1 + 7 * i % 48 for i in range(300)]),
                                      ([20, 3, 48, 0, 9], [48, 3, 48, 12, 40]), ([100, 1, 112, 64], [100, 50, 112, 112])])
def test_tables_no_longer_than_a_unit(dev, new, lens):
    """No sequence can be longer than a unit of positions, so no item is divided and nothing is joined."""
    _paged_case(dev, new, lens, 8, 2, 64, 16, _dt("f16"), _dt("f32"), len(new))
    _paged_case(dev, new, lens, 8, 2, 128, 16, _dt("bf16"), _dt("bf16"), len(new) + 1)


@pytest.mark.parametrize("max_new", [1, 24, None])
def test_pages_behind_32_bits_of_elements(dev, max_new):
    """A pool of 2.7e9 elements, its last pages in use: the writer and the attention reach them."""
    import torch
    from jitllm_b200 import PagedKV
    hkv, d, page_len, pages = 8, 128, 64, 41000
    k = torch.zeros(pages, hkv, page_len, d, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    n = {1: 1, 24: 24, None: 70}[max_new]
    table = torch.tensor([[pages - 1, 3, pages - 2, 32768]], dtype=torch.int32, device="cuda")
    kv, cos, sin = PagedKV(k, v, table), *_tables(256, d)
    qkv = torch.randn(200, (16 + 2 * hkv) * d, device="cuda")
    st, scratch = torch.cuda.current_stream().cuda_stream, _scratch(dev)
    q = torch.empty(200, 16, d, device="cuda", dtype=torch.bfloat16)
    dev.RopeAppend(q, qkv, kv, _starts([200]), torch.tensor([200], dtype=torch.int32, device="cuda"), cos, sin, stream=st)
    out = torch.empty(n, 16, d, device="cuda")
    dev.AttnPaged(out, q[200 - n:].contiguous(), kv, _starts([n]), torch.tensor([200], dtype=torch.int32, device="cuda"), scratch, max_new=max_new,
                  stream=st)
    torch.cuda.synchronize()
    x = qkv.view(200, 16 + 2 * hkv, d)
    vv = x[:, 16 + hkv:].to(torch.bfloat16)
    for p in (0, 63, 64, 128, 199):
        assert torch.equal(v[int(table[0, p // 64]), :, p % 64], vv[p])
    used = sorted(table[0].tolist())
    assert int((v.view(pages, -1).any(1)).sum()) == 4 and v.view(pages, -1).any(1).nonzero().flatten().tolist() == used
    kk = k[table[0].long()].transpose(1, 2).reshape(-1, hkv, d)[:200]                     # as the writer rounded them
    ref, mag, size = _reference(q[200 - n:], kk, vv, 200 - n, d ** -0.5)
    _check(out, ref, mag, size, torch.bfloat16, 200, d)


def test_calls_side_by_side(dev):
    """Calls on two streams, each with its own scratch, in graphs that are replayed at the same time: the bits of one call alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(21)
    lens = [900, 33, 4000, 1, 257]
    pool = Pool(lens, 2, 64, 32, _dt("bf16"), 22)
    work = []
    for new in ([1] * 5, [40, 3, 300, 1, 9], [5] * 3 + [1, 5], [1] * 5):
        q = torch.randn(sum(new), 8, 64, generator=g, device="cuda").bfloat16()
        out = torch.zeros_like(q)
        args = (out, q, pool.kv, _starts(new), torch.tensor(lens, dtype=torch.int32, device="cuda"), _scratch(dev))
        dev.AttnPaged(*args, max_new=max(new), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            dev.AttnPaged(*args, max_new=max(new), stream=stream.cuda_stream)
        work.append((out, out.clone(), args, stream, graph))
    for out, *_ in work:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for _, _, _, stream, graph in work:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone) for out, alone, *_ in work) and dev.StatusPoll()


def test_sequences_may_share_pages(dev):
    import torch
    pool = Pool([200, 200], 2, 64, 32, _dt("f16"), 2)
    pool.table[1, :6] = pool.table[0, :6]                                # a prefix of 192 positions
    k, v = pool.rows[0]
    k1, v1 = torch.cat([k[:192], pool.rows[1][0][192:]]), torch.cat([v[:192], pool.rows[1][1][192:]])
    q = torch.randn(2, 4, 64, device="cuda").half()
    out = torch.empty(2, 4, 64, device="cuda")
    dev.AttnPaged(out, q, pool.kv, _starts([1, 1]), torch.tensor([200, 200], dtype=torch.int32, device="cuda"), _scratch(dev), max_new=1,
                  stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for s, (kk, vv) in enumerate(((k, v), (k1, v1))):
        ref, mag, size = _reference(q[s:s + 1], kk, vv, 199, 64 ** -0.5)
        _check(out[s:s + 1], ref, mag, size, _dt("f16"), 200, 64)


@pytest.mark.parametrize("new,max_new", [([1, 1, 1], 1), ([40, 1, 300], None)])
def test_paged_replays_in_a_graph_on_other_lengths(dev, new, max_new):
    """A captured call follows the tables on the device; two graphs with a scratch each run side by side on two streams."""
    import torch
    lens = [700, 1200, 300]
    pool = Pool([800, 1300, 400], 2, 128, 16, _dt("bf16"), 4)
    total = sum(new)
    runs = []
    for i in range(2):
        q = torch.randn(total, 8, 128, device="cuda").bfloat16()
        out = torch.zeros(total, 8, 128, device="cuda", dtype=torch.bfloat16)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        scratch, starts = _scratch(dev), _starts(new)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            dev.AttnPaged(out, q, pool.kv, starts, ln, scratch, max_new=max_new, stream=side.cuda_stream)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dev.AttnPaged(out, q, pool.kv, starts, ln, scratch, max_new=max_new, stream=torch.cuda.current_stream().cuda_stream)
        runs.append((q, out, ln, scratch, starts, side, graph))
    torch.cuda.synchronize()
    for add in (0, 90):
        for i, (q, out, ln, _, _, side, graph) in enumerate(runs):
            with torch.cuda.stream(side):
                out.zero_()
                ln.copy_(torch.tensor([n + add + i for n in lens], dtype=torch.int32, device="cuda"))
                graph.replay()
        torch.cuda.synchronize()
        for i, (q, out, ln, *_rest) in enumerate(runs):
            at = 0
            for s, n in enumerate(new):
                length = lens[s] + add + i
                k, v = pool.rows[s]
                ref, mag, size = _reference(q[at:at + n], k[:length], v[:length], length - n, 128 ** -0.5)
                _check(out[at:at + n], ref, mag, size, _dt("bf16"), length, 128)
                at += n


# ---------------------------------------------------------------- packed prompts

def _prompt_case(dev, new, hq, hkv, d, dt, out_dt, seed, layout="rows", scale=None, pad=3):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(new)
    total = rows + pad
    nan = torch.full((pad, 1, 1), float("nan"), device="cuda")

    def randn(h):
        return torch.randn(total, h, d, generator=g, device="cuda")
    q, k, v = randn(hq), randn(hkv), randn(hkv)
    k[rows:], v[rows:] = nan, nan                                        # nobody's rows
    if layout == "fused":
        q, k, v = torch.cat([q, k, v], 1).to(dt).split([hq, hkv, hkv], 1)
    else:
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if layout == "cache":
        k, v = (torch.cat([x.transpose(0, 1), torch.full((hkv, 40, d), float("nan"), device="cuda", dtype=dt)], 1)[:, :total].transpose(0, 1)
                for x in (k, v))
    out = torch.full((total, hq, d), 7.0, device="cuda", dtype=out_dt)
    dev.AttnPrompt(out, q, k, v, _starts(new), _scratch(dev), scale=scale, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert dev.StatusPoll()
    assert bool((out[rows:] == 7.0).all())
    at = 0
    for n in new:
        ref, mag, size = _reference(q[at:at + n], k[at:at + n], v[at:at + n], 0, d ** -0.5 if scale is None else scale)
        _check(out[at:at + n], ref, mag, size, dt, n, d)
        at += n
    return out


@pytest.mark.parametrize("dt,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (4, 4, 64), (9, 3, 128), (16, 1, 64), (10, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("layout", ["rows", "fused", "cache"])
def test_prompts_packed(dev, dt, out, hq, hkv, d, layout):
    _prompt_case(dev, [1, 0, 2, 17, 64, 65, 0, 127, 128, 129, 300, 3], hq, hkv, d, _dt(dt), _dt(out), 1 + hq, layout)


@pytest.mark.parametrize("n", [1, 7, 31, 32, 33, 63, 64, 100, 255, 256, 257, 1000, 1531])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (2, 2)])
def test_prompt_of_one_sequence(dev, n, hq, hkv):
    _prompt_case(dev, [n], hq, hkv, 128, _dt("bf16"), _dt("bf16"), n, "cache", pad=0)


def test_long_prompt(dev):
    a = _prompt_case(dev, [6001], 4, 1, 128, _dt("bf16"), _dt("bf16"), 3)
    b = _prompt_case(dev, [6001], 4, 1, 128, _dt("bf16"), _dt("bf16"), 3)
    assert bool((a == b).all())
    _prompt_case(dev, [2500, 1, 4000], 2, 1, 64, _dt("f16"), _dt("f32"), 4, "fused", scale=1.7)


def test_prompts_do_not_reach_one_another(dev):
    """A sequence of NaN between two others; and infinite or NaN values of later positions leave earlier rows alone."""
    import torch
    new = [70, 40, 200]
    q, k, v = (torch.randn(310, h, 128, device="cuda").bfloat16() for h in (8, 2, 2))
    k[70:110], v[70:110] = float("nan"), float("nan")
    k[210, :, 3], v[210, 0, 1], v[211, 1, 77] = float("nan"), float("nan"), float("inf")
    out = torch.zeros(310, 8, 128, device="cuda", dtype=torch.bfloat16)
    dev.AttnPrompt(out, q, k, v, _starts(new), _scratch(dev), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for a, b, n in ((0, 70, 70), (110, 210, 100)):
        ref, mag, size = _reference(q[a:b], k[a:b], v[a:b], 0, 128 ** -0.5)
        _check(out[a:b], ref, mag, size, _dt("bf16"), n, 128)
    assert bool(out[70:110].isnan().all()) and not bool(out[210:].isfinite().all(-1).any())


def test_starts_out_of_order_stay_inside(dev):
    """Falling, negative or too large starts are no sequence's rows: nothing outside [0, total) is touched and the call returns."""
    import torch
    q, k, v = (torch.randn(40, h, 64, device="cuda").half() for h in (4, 2, 2))
    guard = torch.full((42, 4, 64), 7.0, device="cuda")
    out = guard[1:41]
    for starts in ([5, 2, 9, -4, 3], [-7, 1000, 4], [0, 1 << 30]):
        dev.AttnPrompt(out, q, k, v, torch.tensor(starts, dtype=torch.int32, device="cuda"), _scratch(dev),
                       stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert dev.StatusPoll() and bool((guard[0] == 7).all()) and bool((guard[41] == 7).all())


# ---------------------------------------------------------------- the writer, and the three together

def _rot(x, cos, sin):
    import torch
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    c, s = cos[:, None, :].double(), sin[:, None, :].double()
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _tables(n, d):
    import torch
    inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, device="cuda").double() / d))
    ang = torch.arange(n, device="cuda").double()[:, None] * inv[None, :]
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hq,hkv,d,page_len", [(32, 8, 128, 16), (3, 1, 64, 128), (5, 5, 128, 32)])
def test_rope_append(dev, x, dt, hq, hkv, d, page_len):
    import torch
    lens, new = [1, 200, 64, 0, 33, 130], [1, 7, 0, 0, 33, 129]
    pool = Pool(lens, hkv, d, page_len, _dt(dt), 3)
    k0, v0 = pool.k.clone(), pool.v.clone()
    total = sum(new) + 2
    cos, sin = _tables(201, d)
    qkv = torch.randn(total, (hq + 2 * hkv) * d, device="cuda").to(_dt(x))
    q = torch.full((total, hq, d), 7.0, device="cuda", dtype=_dt(dt))
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dev.RopeAppend(q, qkv, pool.kv, _starts(new), lens_d, cos, sin, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((q[sum(new):] == 7.0).all())
    # one rounding to the cache's type of an f32 result: two products and a sum, each off by 2^-24 of at most |a| + |b|
    at, h = 0, _half_step(_dt(dt))
    for s, n in enumerate(new):
        pos = torch.arange(lens[s] - n, lens[s], device="cuda")
        r = qkv[at:at + n].float().view(n, hq + 2 * hkv, d)
        rot = _rot(r[:, :hq + hkv], cos[pos], sin[pos])
        size = (r[:, :hq + hkv].abs().unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1)).double()
        page = pool.table[s].long()[pos // page_len]
        k, v = pool.k[page, :, pos % page_len], pool.v[page, :, pos % page_len]
        for got, ref, sz in ((q[at:at + n], rot[:, :hq], size[:, :hq]), (k, rot[:, hq:], size[:, hq:])):
            err = (got.double() - ref).abs() - (ref.abs() * h + sz * 3 * 2.0 ** -24 * (1 + h) + torch.finfo(_dt(dt)).smallest_normal * h)
            assert not bool((err > 0).any())
        assert torch.equal(v, r[:, hq + hkv:].to(_dt(dt)))
        k0[page, :, pos % page_len], v0[page, :, pos % page_len] = k, v
        at += n
    same = lambda a, b: bool(((a == b) | (a.isnan() & b.isnan())).all())
    assert same(pool.k, k0) and same(pool.v, v0)                         # nothing else was written


def test_rope_append_leaves_out_what_has_no_place(dev):
    """Positions below zero, beyond the rotation's tables or the page table: the row is left out; a bad page takes no k and v."""
    import torch
    pool = Pool([40, 40, 40, 40], 1, 64, 16, _dt("bf16"), 3, spare=0)
    pool.table[2, 2] = pool.k.shape[0]
    k0 = pool.k.clone()
    cos, sin = _tables(48, 64)
    qkv = torch.randn(8, 3 * 64, device="cuda")
    q = torch.full((8, 1, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    lens = torch.tensor([1, 49, 40, 3000000], dtype=torch.int32, device="cuda")     # new rows: 2 each
    dev.RopeAppend(q, qkv, pool.kv, _starts([2, 2, 2, 2]), lens, cos, sin, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    left = (q == 7.0).all(-1).all(-1).tolist()
    assert left == [True, False, False, True, False, False, True, True]
    changed = ((pool.k != k0) & ~(pool.k.isnan() & k0.isnan())).any(-1).any(1)      # [pages][slots]
    want = torch.zeros_like(changed)
    want[int(pool.table[0, 0]), 0] = True                                            # position 0 of the first sequence
    want[int(pool.table[1, 2]), 15] = True                                           # position 47 of the second
    assert torch.equal(changed, want)


@pytest.mark.parametrize("page_len", [16, 128])
def test_append_and_attention_together(dev, page_len):
    """Requests of different lengths in one pool: a packed prompt, a chunk, then single tokens, every step through the writer and the
    paged attention; each request's results are those of one prompt attention over all of its tokens."""
    import torch
    hq, hkv, d, dt = 8, 2, 128, torch.bfloat16
    lens = [150, 21, 300]
    pool = Pool([n + 4 for n in lens], hkv, d, page_len, dt, 6)
    pool.k.fill_(float("nan"))
    pool.v.fill_(float("nan"))
    st = torch.cuda.current_stream().cuda_stream
    cos, sin = _tables(400, d)
    rows = [torch.randn(n + 4, (hq + 2 * hkv) * d, device="cuda") for n in lens]
    got = [[] for _ in lens]
    done, scratch = [0, 0, 0], _scratch(dev)
    for new in ([100, 21, 300], [50, 1, 0], [1, 1, 1], [0, 2, 1], [3, 0, 2]):
        starts = _starts(new)
        lens_d = torch.tensor([a + b for a, b in zip(done, new)], dtype=torch.int32, device="cuda")
        qkv = torch.cat([r[a:a + b] for r, a, b in zip(rows, done, new)])
        q = torch.empty(sum(new), hq, d, device="cuda", dtype=dt)
        out = torch.empty(sum(new), hq, d, device="cuda")
        dev.RopeAppend(q, qkv, pool.kv, starts, lens_d, cos, sin, stream=st)
        dev.AttnPaged(out, q, pool.kv, starts, lens_d, scratch, max_new=max(new), stream=st)
        at = 0
        for s, n in enumerate(new):
            got[s].append(out[at:at + n])
            at += n
        done = [a + b for a, b in zip(done, new)]
    torch.cuda.synchronize()
    assert dev.StatusPoll() and done == [n + 4 for n in lens]
    for s, r in enumerate(rows):
        n = r.shape[0]
        x = r.view(n, hq + 2 * hkv, d)
        page = pool.table[s].long()[torch.arange(n, device="cuda") // page_len]
        slot = torch.arange(n, device="cuda") % page_len
        q = torch.empty(n, hq, d, device="cuda", dtype=dt)
        one = Pool([n], hkv, d, page_len, dt, 1)
        dev.RopeAppend(q, r, one.kv, _starts([n]), torch.tensor([n], dtype=torch.int32, device="cuda"), cos, sin, stream=st)
        k, v = pool.k[page, :, slot], pool.v[page, :, slot]
        assert torch.equal(v, x[:, hq + hkv:].to(dt))
        ref, mag, size = _reference(q, k, v, 0, d ** -0.5)
        _check(torch.cat(got[s]), ref, mag, size, dt, n, d)
        out = torch.empty(n, hq, d, device="cuda")
        dev.AttnPrompt(out, q, k.contiguous(), v.contiguous(), _starts([n]), scratch, stream=st)
        torch.cuda.synchronize()
        _check(out, ref, mag, size, dt, n, d)


def test_refusals(dev):
    import torch
    from jitllm_b200 import DeviceError, PagedKV, _lib
    q, kv = torch.zeros(4, 8, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 2, 128, device="cuda", dtype=torch.bfloat16)
    out, st, scr = torch.empty_like(q), _starts([4]), _scratch(dev)
    dev.AttnPrompt(out, q, kv, kv, st, scr)
    with pytest.raises(ValueError):
        dev.AttnPrompt(out, q, kv.half(), kv.half(), st, scr)            # mixed types
    with pytest.raises(ValueError):
        dev.AttnPrompt(out.cpu(), q, kv, kv, st, scr)                    # not on the device
    with pytest.raises(ValueError):
        dev.AttnPrompt(out, q, kv, kv, st.long(), scr)
    with pytest.raises(ValueError):
        dev.AttnPrompt(out[:3], q, kv, kv, st, scr)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(DeviceError) as e:
            dev.AttnPrompt(out, q, kv, kv, st, scr, **bad)
        assert e.value.status == _lib.EINVAL
    with pytest.raises(DeviceError):
        dev.AttnPrompt(out, q, kv, kv, st, scr[:1000])                   # too little scratch
    with pytest.raises(DeviceError):
        dev.AttnPrompt(out, q, kv, kv, st, scr[1:])                      # misaligned
    z = torch.zeros(4, 34, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(DeviceError) as e:
        dev.AttnPrompt(torch.empty_like(z), z, kv, kv, st, scr)          # 17 heads to one
    assert e.value.status == _lib.ENOTSUP
    y = torch.zeros(4, 3, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(DeviceError):
        dev.AttnPrompt(torch.empty_like(y), y, kv, kv, st, scr)          # 3 over 2
    w = torch.zeros(4, 2, 96, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(DeviceError) as e:
        dev.AttnPrompt(torch.empty_like(w), w, w, w, st, scr)
    assert e.value.status == _lib.ENOTSUP
    big = torch.zeros(4, 2, 132, device="cuda", dtype=torch.bfloat16)[:, :, :128]
    with pytest.raises(DeviceError):
        dev.AttnPrompt(torch.empty(4, 2, 128, device="cuda", dtype=torch.bfloat16), big, kv, kv, st, scr)    # strides of 4
    table, lens = torch.zeros(1, 4, device="cuda", dtype=torch.int32), torch.tensor([4], device="cuda", dtype=torch.int32)
    for page_len in (8, 24, 2048):
        p = torch.zeros(2, 2, page_len, 128, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(DeviceError) as e:
            dev.AttnPaged(out, q, PagedKV(p, p, table), st, lens, scr)
        assert e.value.status == _lib.ENOTSUP
    p = torch.zeros(2, 2, 16, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        PagedKV(p.float(), p.float(), table)
    with pytest.raises(ValueError):
        PagedKV(p, p, table.long())
    pk = PagedKV(p, p.clone(), table)
    with pytest.raises(DeviceError):
        dev.AttnPaged(out, q, pk, st, lens, scr, max_new=0)
    with pytest.raises(ValueError):
        dev.AttnPaged(out, q, pk, st, lens[:0], scr)
    cos = torch.zeros(8, 64, device="cuda")
    with pytest.raises(ValueError):
        dev.RopeAppend(q, torch.zeros(4, 11 * 128, device="cuda"), pk, st, lens, cos, cos)
    with pytest.raises(ValueError):
        dev.RopeAppend(q, torch.zeros(4, 12 * 128, device="cuda"), pk, st, lens, cos.double(), cos.double())
    torch.cuda.synchronize()
    # nothing to do is no error
    dev.AttnPrompt(out[:0], q[:0], kv[:0], kv[:0], st, scr)
    dev.AttnPaged(out[:0], q[:0], pk, st, lens, scr)


def test_the_callers_device_stays_current(dev):
    import torch
    q, kv = torch.zeros(4, 8, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 2, 128, device="cuda", dtype=torch.bfloat16)
    before, launches = torch.cuda.current_device(), dev.Stats().launches
    dev.AttnPrompt(torch.empty_like(q), q, kv, kv, _starts([4]), _scratch(dev))
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before and dev.Stats().launches > launches
