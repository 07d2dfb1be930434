"""The decoder's serving calls at the edges of what they allow: rows that are nobody's, prompts and contexts longer than the tables."""
import pytest

pytestmark = pytest.mark.gpu


def _decoder(dev, max_len=256, max_prefill=512):
    from jitllm_b200.decoder import Config, Decoder
    cfg = Config(n_layer=2, hidden=512, n_head=4, n_kv=2, head_dim=128, ffn=1024, vocab=2048)
    return Decoder(dev, cfg, max_batch=3, max_len=max_len, max_prefill=max_prefill, seed=11)


def _i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return _i32(at)


def _tokens(n, seed):
    import torch
    return torch.randint(0, 2048, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("new,rows", [([100], 512), ([30, 0, 7], 300), ([300], 300), ([10, 400], 500)])
def test_packed_scores_do_not_depend_on_the_tables(dev, new, rows):
    """Rows behind the last prompt and prompts longer than max_len: the bits of a decoder whose tables hold every position."""
    import torch
    tokens, starts, got = _tokens(rows, 5), _starts(new), []
    with torch.no_grad():
        for max_len in (64, 512):
            dec = _decoder(dev, max_len)
            nxt = dec.score_packed(tokens, starts)
            got.append((nxt, dec.last_logits.clone()))
        torch.cuda.synchronize()
    live = [s for s, n in enumerate(new) if n]
    assert bool(got[0][1][live].isfinite().all())
    assert torch.equal(got[0][1][live], got[1][1][live]) and torch.equal(got[0][0][live], got[1][0][live])
    assert dev.StatusPoll()


def test_starts_behind_the_rows_index_none(dev):
    """A last sequence that claims more rows than there are: the others' results, and no index out of range."""
    import torch
    dec = _decoder(dev)
    dec.open_pool(40, 16)
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    tokens = _tokens(40, 6)
    with torch.no_grad():
        dec.score_packed(tokens, _starts([20, 20]))
        want = dec.last_logits[0].clone()
        dec.score_packed(tokens, _i32([0, 20, 900]))
        assert torch.equal(dec.last_logits[0], want)
        dec.step_paged(tokens, _starts([20, 20]), _i32([20, 20]), table, 20)
        want = dec.last_logits[0].clone()
        dec.step_paged(tokens, _i32([0, 20, 900]), _i32([20, 20]), table, 20)
        assert torch.equal(dec.last_logits[0], want)
        torch.cuda.synchronize()
    assert dev.StatusPoll()


def test_a_captured_step_keeps_its_scratch(dev):
    """Scores captured before the pool is opened (again), replayed after it while other tensors come and go: the same bits, and nobody
    else's memory is written."""
    import torch
    dec = _decoder(dev)
    rows, starts = _tokens(300, 7), _starts([200, 100])
    with torch.no_grad():
        dec.score_packed(rows, starts)
        want = dec.last_logits.clone()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            dec.score_packed(rows, starts)
            logits = dec.last_logits
        for _ in range(2):
            dec.open_pool(40, 16)
            guard = [torch.full((dev.AttnScratchBytes(),), 7, device="cuda", dtype=torch.uint8) for _ in range(3)]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits, want) and all(bool((g == 7).all()) for g in guard)
    assert dev.StatusPoll()
    graph.reset()


def test_no_two_steps_have_one_scratch(dev):
    """Two captured steps, an eager one on another stream and one on this: none has the scratch of another that is still to run."""
    import torch
    dec = _decoder(dev)
    dec.open_pool(40, 16)
    at, real = [], dec._attn_scratch

    def watched():
        at.append(real())
        return at[-1]
    dec._attn_scratch = watched
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    args = (_tokens(2, 8), _starts([1, 1]), _i32([1, 1]), table, 1)
    graphs = []
    with torch.no_grad():
        dec.step_paged(*args)
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            torch.cuda.synchronize()
            with torch.cuda.graph(graphs[-1]):
                dec.step_paged(*args)
        with torch.cuda.stream(torch.cuda.Stream()):
            dec.step_paged(*args)
        torch.cuda.synchronize()
    assert len({t.data_ptr() for t in at}) == 4
    for g in graphs:
        g.reset()


@pytest.mark.parametrize("new,lens", [([1], [65]), ([1, 1, 1], [64, 65, 30]), ([2, 1, 2], [66, 90, 64]), ([12, 3, 1], [70, 40, 64]), ([40, 1, 20], [100, 10, 20])])
def test_positions_behind_the_tables_are_not_numbers(dev, new, lens):
    """A request that grows past max_len while its pages go on: NaN logits and the token -1 instead of a plausible one; the requests beside it
    have the bits of a decoder whose tables go on, too."""
    import torch
    got = []
    full = [_tokens(n, 20 + i) for i, n in enumerate(lens)]
    with torch.no_grad():
        for max_len in (64, 512):
            dec = _decoder(dev, max_len)
            dec.open_pool(24, 16)
            table = torch.arange(24, device="cuda", dtype=torch.int32).view(3, 8)[:len(lens)].contiguous()
            dec.k_pool.normal_(generator=torch.Generator(device="cuda").manual_seed(1))      # what an earlier owner of the pages left
            dec.v_pool.normal_(generator=torch.Generator(device="cuda").manual_seed(2))
            if any(n > m for n, m in zip(lens, new)):
                rest = [n - m for n, m in zip(lens, new)]
                dec.step_paged(torch.cat([f[:r] for f, r in zip(full, rest)]), _starts(rest), _i32(rest), table, max(rest))
            junk = [torch.randn(1 << k, device="cuda") for k in (10, 14, 17, 20)]            # what the step's tensors get
            torch.cuda.synchronize()
            del junk
            nxt = dec.step_paged(torch.cat([f[n - m:] for f, n, m in zip(full, lens, new)]), _starts(new), _i32(lens), table, max(new))
            got.append((nxt.tolist(), dec.last_logits.clone()))
        torch.cuda.synchronize()
    for s, n in enumerate(lens):
        if n > 64:
            assert bool(got[0][1][s].isnan().all()) and got[0][0][s] == -1
        else:
            assert torch.equal(got[0][1][s], got[1][1][s]) and got[0][0][s] == got[1][0][s] >= 0
        assert bool(got[1][1][s].isfinite().all())
    assert dev.StatusPoll()


@pytest.mark.parametrize("rows", [1, 2, 12])
def test_a_bad_page_has_no_next_token(dev, rows):
    import torch
    dec = _decoder(dev)
    dec.open_pool(8, 16)
    table = torch.tensor([[0, 1], [2, 99]], device="cuda", dtype=torch.int32)
    tokens = _tokens(2 * rows, 30)
    with torch.no_grad():
        nxt = dec.step_paged(tokens, _starts([rows, rows]), _i32([20, 20]), table, rows)
        torch.cuda.synchronize()
    assert nxt[0].item() >= 0 and nxt[1].item() == -1 and bool(dec.last_logits[0].isfinite().all())
