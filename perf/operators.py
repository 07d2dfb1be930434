"""Timed cases of the operators that serve several requests at once, over the library's public entry points.

Kinds of case (the "kind" of each dict):

  prompt   Device.AttnPrompt: causal attention over packed prompts of different lengths, grouped query heads.
  paged    Device.AttnPaged: attention of each sequence's new tokens (one, a handful, a chunk) over a cache in pages.
  append   Device.RopeAppend: RoPE of the projected rows, k and v written to the sequences' pages.

With `own` false `run` computes the same in elementary torch operations, in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SCORES = 1 << 28          # the plain forms' scores at a time


def listed():
    return [
        # the smallest prompt, where launch and latency are the time: a one-line question, 32 heads over 8
        dict(name="prompt_7", kind="prompt", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, nseq=1, lo=7, hi=7, layout="rows"),
        # one ragged prompt, k and v in a contiguous per-sequence cache
        dict(name="prompt_1531", kind="prompt", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, nseq=1, lo=1531, hi=1531, layout="cache"),
        # prompts of many requests packed, from one token to pages of text; small heads, q, k and v inside the projection's rows
        dict(name="prompts_24_packed", kind="prompt", dtype="f16", out="f16", hq=16, hkv=2, d=64, nseq=24, lo=1, hi=1900, layout="fused"),
        # a long document: the largest
        dict(name="prompt_16384", kind="prompt", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, nseq=1, lo=16384, hi=16384, layout="rows"),
        # decode of one sequence, the latency of a single user
        dict(name="decode_1x2049", kind="paged", dtype="bf16", out="f32", hq=32, hkv=8, d=128, page_len=16, nseq=1, lo=2049, hi=2049,
             new=1, chunks=0, chunk=0),
        # batched decode, contexts of all lengths
        dict(name="decode_64_ragged", kind="paged", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, page_len=64, nseq=64, lo=37, hi=8200,
             new=1, chunks=0, chunk=0),
        # one long context: the cache's axis is all the parallelism there is
        dict(name="decode_1x131071", kind="paged", dtype="f16", out="f32", hq=16, hkv=2, d=128, page_len=256, nseq=1, lo=131071, hi=131071,
             new=1, chunks=0, chunk=0),
        # a few tokens to verify for each of many sequences
        dict(name="verify_32x5", kind="paged", dtype="bf16", out="bf16", hq=64, hkv=8, d=64, page_len=32, nseq=32, lo=300, hi=4100,
             new=5, chunks=0, chunk=0),
        # a prompt's later chunk over what is cached already
        dict(name="chunk_1000_at_17000", kind="paged", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, page_len=16, nseq=1, lo=17000, hi=17000,
             new=1000, chunks=0, chunk=0),
        # a serving step: single tokens of most sequences, chunks of two
        dict(name="step_26_mixed", kind="paged", dtype="bf16", out="bf16", hq=32, hkv=8, d=128, page_len=64, nseq=26, lo=900, hi=6000,
             new=1, chunks=2, chunk=501),
        # the cache's writer beside them: a decode step and a prompt's chunk
        dict(name="append_64", kind="append", dtype="bf16", x="f32", hq=32, hkv=8, d=128, page_len=64, nseq=64, lo=37, hi=2049,
             new=1, chunks=0, chunk=0),
        dict(name="append_4096", kind="append", dtype="bf16", x="f32", hq=32, hkv=8, d=128, page_len=16, nseq=3, lo=1400, hi=5001,
             new=1365, chunks=0, chunk=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8])
    return hkv * rng.choice([1, 2, 3, 4, 5, 8]), hkv


def draw(rng):
    kind = rng.choices(["prompt", "paged", "append"], [3, 5, 1])[0]
    hq, hkv = _heads(rng)
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), hq=hq, hkv=hkv, d=rng.choice([64, 128, 128]))
    if kind == "prompt":
        c["out"] = rng.choice([c["dtype"], c["dtype"], "f32"])
        c["nseq"] = rng.choice([1, 1, 2, _log(rng, 3, 40)])
        c["hi"] = _log(rng, 1, 12000 if c["nseq"] <= 2 else 2500)
        while 4 * c["d"] * hq * c["nseq"] * c["hi"] ** 2 > 4e12:      # no more than the largest listed case
            c["hi"] = c["hi"] * 2 // 3
        c["lo"] = _log(rng, 1, c["hi"]) if c["nseq"] > 1 else c["hi"]
        c["layout"] = rng.choice(["rows", "fused"] + (["cache"] if c["nseq"] == 1 else []))
        return c
    c["page_len"] = rng.choice([16, 16, 32, 64, 128, 256])
    c["nseq"] = rng.choice([1, 2, _log(rng, 3, 100)])
    c["hi"] = _log(rng, 1, 120000 // c["nseq"] + 600)
    c["lo"] = _log(rng, 1, c["hi"]) if c["nseq"] > 1 else c["hi"]
    c["new"] = rng.choice([1, 1, 1, _log(rng, 2, 9), _log(rng, 9, 700)])
    c["chunks"] = rng.choice([0, 0, 1, 2]) if c["nseq"] > 2 else 0
    c["chunk"] = _log(rng, 9, 1200) if c["chunks"] else 0
    if kind == "append":
        c["x"] = rng.choice(["f32", "f32", "bf16", "f16"])
    else:
        c["out"] = rng.choice([c["dtype"], "f32"])
    return c


def _spread(n, lo, hi):
    """n lengths from lo to hi, even over their logarithm, in an order that mixes them."""
    at = [int(round(lo * (hi / lo) ** (i / (n - 1)))) if n > 1 else hi for i in range(n)]
    step = next(s for s in range(max(1, n // 3), 2 * n + 2) if math.gcd(s, n) == 1)
    return [at[i * step % n] for i in range(n)]


def _lengths(case):
    """(positions of each sequence, its new tokens among them)."""
    lens = _spread(case["nseq"], case["lo"], case["hi"])
    if case["kind"] == "prompt":
        return lens, lens
    new = [min(case["chunk"] if i < case["chunks"] else case["new"], n) for i, n in enumerate(lens)]
    return lens, new


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def _inputs(case, seed):
    """The tensors of a case, from the seed alone: what prepare and exact both start from."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, new = _lengths(case)
    starts = _starts(new)
    rows, hq, hkv, d, dt = starts[-1], case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # heads differ in how sharply they attend
    sharp = torch.exp2(torch.rand(hq, generator=g, device="cuda") * 3 - 1)
    t = dict(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["kind"] == "prompt":
        if case["layout"] == "fused":
            t["q"], t["k"], t["v"] = randn(rows, hq + 2 * hkv, d).to(dt).split([hq, hkv, hkv], dim=1)
        elif case["layout"] == "cache":
            t["q"] = randn(rows, hq, d).to(dt)
            t["k"], t["v"] = (randn(hkv, rows + 33, d).to(dt)[:, :rows].transpose(0, 1) for _ in range(2))
        else:
            t["q"], t["k"], t["v"] = randn(rows, hq, d).to(dt), randn(rows, hkv, d).to(dt), randn(rows, hkv, d).to(dt)
        t["q"].mul_(sharp[:, None].to(dt))
        return t
    p = case["page_len"]
    npages = [(n + p - 1) // p for n in lens]
    pool = sum(npages) + max(2, sum(npages) // 8)                 # some pages belong to nobody
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(npages) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(npages):
        table[s, :n] = order[at:at + n]
        at += n
    t.update(table=table, k=randn(pool, hkv, p, d).to(dt), v=randn(pool, hkv, p, d).to(dt))
    if case["kind"] == "paged":
        t["q"] = (randn(rows, hq, d) * sharp[:, None]).to(dt)
    else:
        t["qkv"] = randn(rows, (hq + 2 * hkv) * d).to(DTYPES[case["x"]])
        inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, device="cuda").double() / d))
        ang = torch.arange(max(lens), device="cuda").double()[:, None] * inv[None, :]
        t["cos"], t["sin"] = ang.cos().float(), ang.sin().float()
    return t


_device = None


def _dev():
    global _device
    if _device is None:
        from jitllm_b200 import Device
        _device = Device(0)
    return _device


def prepare(case, seed):
    t = _inputs(case, seed)
    rows, d = t["starts"][-1].item(), case["d"]
    lens, new = _lengths(case)
    state = dict(case=case, t=t, lens=lens, new=new, scale=1.0 / math.sqrt(d))
    if case["kind"] == "append":
        state["q_out"] = torch.empty(rows, case["hq"], d, device="cuda", dtype=DTYPES[case["dtype"]])
    else:
        state["out"] = torch.empty(rows, case["hq"], d, device="cuda", dtype=DTYPES[case["out"]])
    if own:
        from jitllm_b200 import PagedKV
        dev = state["dev"] = _dev()
        if case["kind"] != "append":
            state["scratch"] = torch.empty(dev.AttnScratchBytes(), device="cuda", dtype=torch.uint8)
        if case["kind"] != "prompt":
            state["kv"] = PagedKV(t["k"], t["v"], t["table"])
    return state


def run(state):
    case, t = state["case"], state["t"]
    if own:
        return _run_own(state, case, t, torch.cuda.current_stream().cuda_stream)
    return {"prompt": _plain_prompt, "paged": _plain_paged, "append": _plain_append}[case["kind"]](state, case, t)


def _run_own(state, case, t, stream):
    dev = state["dev"]
    if case["kind"] == "prompt":
        dev.AttnPrompt(state["out"], t["q"], t["k"], t["v"], t["starts"], state["scratch"], scale=state["scale"], stream=stream)
        return state["out"]
    if case["kind"] == "paged":
        dev.AttnPaged(state["out"], t["q"], state["kv"], t["starts"], t["lens"], state["scratch"], max_new=max(state["new"]),
                      scale=state["scale"], stream=stream)
        return state["out"]
    dev.RopeAppend(state["q_out"], t["qkv"], state["kv"], t["starts"], t["lens"], t["cos"], t["sin"], stream=stream)
    return state["q_out"], t["k"], t["v"]


# ---------------------------------------------------------------- plain forms

def _attend(out, q, k, v, first, scale):
    """out, q [n][hq][d]; k, v [len][hkv][d]; query i sits at position first + i. In pieces of rows, each piece over the positions
    that any of its rows sees."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    kt, vt = k.float().permute(1, 2, 0), v.float().transpose(0, 1)
    step = max(1, SCORES // (hq * length))
    for a in range(0, n, step):
        b = min(n, a + step)
        seen = min(length, first + b)
        s = q[a:b].float().view(b - a, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d) @ kt[:, :, :seen] * scale
        s = s.view(hkv, hq // hkv, b - a, seen)
        pos = torch.arange(first + a, first + b, device=q.device)
        hidden = torch.arange(seen, device=q.device)[None, :] > pos[:, None]
        s.masked_fill_(hidden, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = (e / e.sum(-1, keepdim=True)).view(hkv, -1, seen) @ vt[:, :seen]
        out[a:b] = o.view(hkv, hq // hkv, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d).to(out.dtype)


def _plain_prompt(state, case, t):
    at = _starts(state["new"])
    for a, b in zip(at, at[1:]):
        _attend(state["out"][a:b], t["q"][a:b], t["k"][a:b], t["v"][a:b], 0, state["scale"])
    return state["out"]


def _plain_paged(state, case, t):
    at, p = _starts(state["new"]), case["page_len"]
    for s, n in enumerate(state["lens"]):
        pages = t["table"][s, :(n + p - 1) // p].long()
        k, v = (x[pages].transpose(1, 2).reshape(-1, case["hkv"], case["d"])[:n] for x in (t["k"], t["v"]))
        a, b = at[s], at[s + 1]
        _attend(state["out"][a:b], t["q"][a:b], k, v, n - (b - a), state["scale"])
    return state["out"]


def _positions(t, rows):
    """(sequence, position) of each new row."""
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(t["starts"][1:].contiguous(), r, right=True)
    return seq, (t["lens"][seq] - t["starts"][seq + 1] + r).long()


def _plain_append(state, case, t):
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page_len"]
    rows = t["qkv"].shape[0]
    seq, pos = _positions(t, rows)
    x = t["qkv"].float().view(rows, hq + 2 * hkv, d)
    c, s = t["cos"][pos][:, None, :], t["sin"][pos][:, None, :]
    a, b = x[:, :hq + hkv, 0::2], x[:, :hq + hkv, 1::2]
    rot = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    page, slot = t["table"][seq, pos // p].long(), pos % p
    state["q_out"].copy_(rot[:, :hq])
    t["k"][page, :, slot] = rot[:, hq:].to(t["k"].dtype)
    t["v"][page, :, slot] = x[:, hq + hkv:].to(t["v"].dtype)
    return state["q_out"], t["k"], t["v"]


# ---------------------------------------------------------------- work and exact values

def _pairs(case):
    lens, new = _lengths(case)
    return sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))


def work(case):
    lens, new = _lengths(case)
    rows, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
    if case["kind"] == "append":
        x = 4 if case["x"] == "f32" else 2
        return {"bytes": rows * ((hq + 2 * hkv) * d * (x + 2) + d * 4 + 8), "flops": rows * (hq + hkv) * d * 3}
    kv = sum(n for n, m in zip(lens, new) if m)
    ob = 4 if case["out"] == "f32" else 2
    return {"bytes": rows * hq * d * (2 + ob) + kv * hkv * d * 4, "flops": 4 * d * hq * _pairs(case)}


def exact(case, seed):
    t = _inputs(case, seed)
    lens, new = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "append":
        return _exact_append(case, t, lens, new)
    out = torch.empty(sum(new), hq, d, device="cuda", dtype=torch.float64)
    row = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        if case["kind"] == "prompt":
            k, v = t["k"][row:row + n].double(), t["v"][row:row + n].double()
        else:
            p = case["page_len"]
            where = torch.arange(n, device="cuda")
            page = t["table"][s].long()[where // p]
            k, v = t["k"][page, :, where % p].double(), t["v"][page, :, where % p].double()
        for h in range(hq):
            kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
            step = max(1, (1 << 27) // n)
            for a in range(0, m, step):
                b = min(m, a + step)
                logits = torch.einsum("id,jd->ij", t["q"][row + a:row + b, h].double(), kh) / d ** 0.5
                last = torch.arange(n - m + a, n - m + b, device="cuda")
                logits = torch.where(torch.arange(n, device="cuda")[None, :] <= last[:, None], logits, -math.inf)
                out[row + a:row + b, h] = torch.softmax(logits, dim=1) @ vh
        row += m
    return out


def _exact_append(case, t, lens, new):
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page_len"]
    k, v = t["k"].double(), t["v"].double()
    q = torch.empty(sum(new), hq, d, device="cuda", dtype=torch.float64)
    row = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        where = torch.arange(n - m, n, device="cuda")
        x = t["qkv"][row:row + m].double().view(m, hq + 2 * hkv, d // 2, 2)
        turn = torch.complex(t["cos"][where].double(), t["sin"][where].double())[:, None, :]
        rot = torch.view_as_real(torch.view_as_complex(x[:, :hq + hkv].contiguous()) * turn).flatten(-2)
        page = t["table"][s].long()[where // p]
        q[row:row + m] = rot[:, :hq]
        k[page, :, where % p] = rot[:, hq:]
        v[page, :, where % p] = x[:, hq + hkv:].flatten(-2)
        row += m
    return q, k, v
