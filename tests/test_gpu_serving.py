"""Requests of different lengths through the decoder at once: step_paged (the pool's writer, the paged attention and the matmul chain
together) and score_packed, against the same requests one at a time.

Both sides round q, k, v and the attention's rows to bf16 at the same places, so they differ by the order of their sums and, where the
token counts differ, by the matmul kernels that take them (each within 2e-3 of float64 by itself, two layers of four and the head): the
decoder's own bar between two of its forms of a step, 1e-2 of the largest logit."""
import pytest

pytestmark = pytest.mark.gpu


def _decoder(dev, head_dim=128, max_len=256):
    from jitllm_b200.decoder import Config, Decoder
    cfg = Config(n_layer=2, hidden=512, n_head=4, n_kv=2, head_dim=head_dim, ffn=1024, vocab=2048)
    return Decoder(dev, cfg, max_batch=3, max_len=max_len, max_prefill=max_len, seed=11)


def _i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return _i32(at)


def _alone(dec, tokens):
    """Logits after `tokens`, one prompt, through prefill."""
    dec.prefill(tokens)
    return dec.last_logits[0].double()


def _near(got, ref):
    assert bool(got.isfinite().all())
    err = float((got.double() - ref).abs().max() / ref.abs().max())
    assert err < 1e-2, err


@pytest.mark.parametrize("head_dim,page_len", [(128, 16), (64, 32)])
def test_requests_share_a_pool(dev, head_dim, page_len):
    import torch
    dec = _decoder(dev, head_dim)
    g = torch.Generator(device="cuda").manual_seed(3)
    full = [torch.randint(0, 2048, (n,), device="cuda", generator=g) for n in (90, 33, 200)]
    per = 256 // page_len
    dec.open_pool(3 * per + 2, page_len)
    table = torch.randperm(3 * per + 2, generator=g, device="cuda")[:3 * per].view(3, per).to(torch.int32)
    done = [0, 0, 0]
    with torch.no_grad():
        # a prompt and a chunk; the rest of it and a late request; single tokens; one idle; a handful
        for new in ([80, 0, 150], [1, 30, 45], [1, 1, 1], [2, 1, 0], [5, 1, 3], [1, 0, 1]):
            rows = torch.cat([f[a:a + b] for f, a, b in zip(full, done, new)])
            done = [a + b for a, b in zip(done, new)]
            nxt = dec.step_paged(rows, _starts(new), _i32(done), table, max(new))
            logits = dec.last_logits.clone()
            assert torch.equal(nxt, logits.argmax(-1))
            for s in range(3):
                if new[s]:
                    _near(logits[s], _alone(dec, full[s][:done[s]]))
        torch.cuda.synchronize()
    assert dev.StatusPoll() and done == [90, 33, 200]


def test_a_captured_step_replays_on_other_lengths(dev):
    """Single tokens of three requests, captured once, replayed as they grow over a page's end."""
    import torch
    dec = _decoder(dev)
    g = torch.Generator(device="cuda").manual_seed(4)
    full = [torch.randint(0, 2048, (n,), device="cuda", generator=g) for n in (20, 40, 60)]
    dec.open_pool(16, 16)
    table = torch.arange(15, device="cuda", dtype=torch.int32).view(3, 5)
    done = [14, 30, 50]
    with torch.no_grad():
        dec.step_paged(torch.cat([f[:n] for f, n in zip(full, done)]), _starts(done), _i32(done), table, 50)
        tok, lens, starts = torch.zeros(3, dtype=torch.int64, device="cuda"), _i32([n + 1 for n in done]), _starts([1, 1, 1])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            tok.copy_(torch.stack([f[n] for f, n in zip(full, done)]))
            dec.step_paged(tok, starts, lens, table, 1)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dec.step_paged(tok, starts, lens, table, 1)
            logits = dec.last_logits
        for _ in range(5):
            tok.copy_(torch.stack([f[n] for f, n in zip(full, done)]))
            done = [n + 1 for n in done]
            lens.copy_(_i32(done))
            graph.replay()
            torch.cuda.synchronize()
            got = logits.clone()
            for s in range(3):
                _near(got[s], _alone(dec, full[s][:done[s]]))
    assert dev.StatusPoll()


def test_packed_prompts_are_scored_as_if_alone(dev):
    import torch
    dec = _decoder(dev)
    g = torch.Generator(device="cuda").manual_seed(5)
    new = [17, 1, 0, 120, 64]
    rows = torch.randint(0, 2048, (sum(new),), device="cuda", generator=g)
    starts = _starts(new)
    with torch.no_grad():
        nxt = dec.score_packed(rows, starts)
        logits = dec.last_logits.clone()
        assert torch.equal(nxt, logits.argmax(-1))
        at = 0
        for s, n in enumerate(new):
            if n:
                _near(logits[s], _alone(dec, rows[at:at + n]))
            at += n
    assert dev.StatusPoll()


@pytest.mark.parametrize("real,pad", [([1, 1, 1], 3), ([30, 1, 5], 12)])
def test_rows_behind_the_last_request_reach_nothing(dev, real, pad):
    """A step of a fixed number of rows, the last of them nobody's: whatever memory they start from, the requests' logits and the pool are
    the same to the bit."""
    import torch
    dec = _decoder(dev)
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = torch.randint(0, 2048, (sum(real) + pad,), device="cuda", generator=g)
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(3, 4)
    got = []
    with torch.no_grad():
        for fill in (0.0, float("nan"), 1e30):
            dec.open_pool(12, 16)
            junk = [torch.full((n,), fill, device="cuda") for n in (1 << 10, 1 << 14, 1 << 17, 1 << 20)]      # what the step's tensors get
            torch.cuda.synchronize()
            del junk
            dec.step_paged(rows, _starts(real), _i32(real), table, max(real))
            got.append((dec.last_logits.clone(), dec.k_pool.clone(), dec.v_pool.clone()))
        torch.cuda.synchronize()
    assert bool(got[0][0].isfinite().all())
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
