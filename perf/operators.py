"""What is measured of the operators at the head end of a step: log probabilities of given tokens (with entropy and top
alternatives) over logits, products with 4-bit weights and group scales, and the head product that returns log
probabilities without writing its logits.  Each case has a plain form in elementary torch operations and, where `own` is
set, the call a user makes of the library."""
import math

import torch

own = False

MASKED = -math.inf


def listed():
    return [
        # one decoded token of a chat reply: its log probability and five alternatives (latency counts)
        dict(name="logprobs-1x65536-top5", op="logprobs", rows=1, vocab=65536, half=False, given=1, top=5, pad=0, masked=False),
        # a batch of 256 sequences, each with the twenty alternatives that an API offers at most
        dict(name="logprobs-256x65536-top20", op="logprobs", rows=256, vocab=65536, half=False, given=1, top=20, pad=0, masked=False),
        # the logits of a 4096-token document kept in 16 bits: perplexity, no alternatives
        dict(name="logprobs-4096x65536-f16", op="logprobs", rows=4096, vocab=65536, half=True, given=1, top=0, pad=0, masked=False),
        # odd vocabulary in rows with a stride of their own, most tokens masked by a grammar, three candidates per row
        dict(name="logprobs-37x32001-masked", op="logprobs", rows=37, vocab=32001, half=False, given=3, top=8, pad=62, masked=True),
        # one token through a square projection, symmetric codes
        dict(name="w4-1x4096x4096-g64-sym", op="w4", rows=1, n=4096, k=4096, group=64, symmetric=True),
        # one token through the head, fine groups
        dict(name="w4-1x65536x4096-g32", op="w4", rows=1, n=65536, k=4096, group=32, symmetric=False),
        # five sequences, an odd number of channels, a last group that is not full
        dict(name="w4-5x2561x10272-g128", op="w4", rows=5, n=2561, k=10272, group=128, symmetric=False),
        # a large decode batch through a channel-mix key
        dict(name="w4-96x10240x2560-g64", op="w4", rows=96, n=10240, k=2560, group=64, symmetric=False),
        # two sequences scored on a 4-bit head
        dict(name="head-2x65536x2048-w4g64", op="head", rows=2, n=65536, k=2048, fmt="w4", group=64),
        # an odd prompt on a narrow model with an 8-bit head and an odd vocabulary
        dict(name="head-77x32003x768-w8", op="head", rows=77, n=32003, k=768, fmt="w8", group=0),
        # one prefill chunk of a prompt that is scored
        dict(name="head-128x65536x4096-f16", op="head", rows=128, n=65536, k=4096, fmt="f16", group=0),
        # a whole document at once
        dict(name="head-2048x65536x4096-f16", op="head", rows=2048, n=65536, k=4096, fmt="f16", group=0),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("logprobs", "w4", "head"))
    if op == "logprobs":
        vocab = _spread(rng, 1000, 131072)
        rows = _spread(rng, 1, min(4096, (1 << 28) // vocab))
        given = rng.choice((1, 1, 2, 3, 4))
        return dict(op=op, rows=rows, vocab=vocab, half=rng.random() < 0.3, given=given, top=rng.choice((0, 1, 5, 8, 20, 32)),
                    pad=rng.choice((0, 0, 1, 7, 64)), masked=rng.random() < 0.3)
    k = 32 * _spread(rng, 8, 512)
    n = _spread(rng, 64, min(65536, (1 << 28) // k))
    if op == "w4":
        rows = _spread(rng, 1, 256)
        return dict(op=op, rows=rows, n=n, k=k, group=rng.choice((32, 64, 128)), symmetric=rng.random() < 0.5)
    rows = _spread(rng, 1, min(2048, max(1, (1 << 38) // (n * k))))
    fmt = rng.choice(("f16", "f16", "w8", "w4"))
    return dict(op=op, rows=rows, n=n, k=k, fmt=fmt, group=rng.choice((32, 64, 128)) if fmt == "w4" else 0)


def work(case):
    rows = case["rows"]
    if case["op"] == "logprobs":
        size = rows * case["vocab"]
        out = rows * (8 + 4 * case["given"] + 8 * case["top"])
        return {"bytes": size * (2 if case["half"] else 4) + rows * 8 * case["given"] + out, "flops": 6.0 * size}
    n, k = case["n"], case["k"]
    fmt = case.get("fmt", "w4")
    if fmt == "w4":
        groups = -(-k // case["group"])
        weight = n * k // 2 + n * groups * (2 if case.get("symmetric") else 4)
    else:
        weight = n * k * (2 if fmt == "f16" else 1) + (2 * n if fmt == "w8" else 0)
    out = rows * n * 2 if case["op"] == "w4" else rows * 20
    return {"bytes": weight + rows * k * 2 + out, "flops": 2.0 * rows * n * k}


def _codes4(n, k, group, symmetric, gen, size):
    q = torch.randint(0, 256, (n, k // 2), device="cuda", dtype=torch.uint8, generator=gen)
    groups = -(-k // group)
    scale = ((0.5 + torch.rand(n, groups, device="cuda", generator=gen)) * size).half()
    zero = None if symmetric else torch.randint(4, 12, (n, groups), device="cuda", generator=gen).half()
    return q, scale, zero


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows = case["rows"]
    s = dict(case)
    if case["op"] == "logprobs":
        vocab, dtype = case["vocab"], torch.float16 if case["half"] else torch.float32
        whole = torch.empty(rows, vocab + case["pad"], device="cuda", dtype=dtype)
        for r in range(0, rows, 512):  # (a part at a time: the draws are made in 32 bits)
            part = torch.randn(min(512, rows - r), vocab, device="cuda", generator=gen) * 2.5 - 4
            if case["masked"]:
                part[torch.rand(part.shape, device="cuda", generator=gen) < 0.9] = MASKED
            whole[r:r + 512, :vocab] = part.to(dtype)
        if case["pad"]:
            whole[:, vocab:] = 1e4  # not part of the rows
        if case["masked"] and rows > 2:
            whole[rows // 2] = MASKED  # a row with nothing left
            whole[rows // 3, 3:] = MASKED  # and one with fewer tokens than alternatives are asked for
        s["logits"] = whole[:, :vocab]
        tokens = torch.randint(0, vocab, (rows, case["given"]), device="cuda", generator=gen)
        tokens[torch.rand(tokens.shape, device="cuda", generator=gen) < 0.1] = -1  # padding of a batch
        s["tokens"] = tokens
        return s
    n, k = case["n"], case["k"]
    s["x"] = torch.randn(rows, k, device="cuda", generator=gen).half()
    size = 1.3 / math.sqrt(k)  # of a weight: logits of about this model's width
    if case["op"] == "w4":
        s["q"], s["scale"], s["zero"] = _codes4(n, k, case["group"], case["symmetric"], gen, size / 4.6)
        return s
    s["zero"] = s["scale"] = None
    if case["fmt"] == "f16":
        s["w"] = torch.empty(n, k, device="cuda", dtype=torch.float16).normal_(0, size, generator=gen)
    elif case["fmt"] == "w8":
        s["w"] = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8, generator=gen)
        s["scale"] = ((0.5 + torch.rand(n, device="cuda", generator=gen)) * (size / 74)).half()
    else:
        s["w"], s["scale"], s["zero"] = _codes4(n, k, case["group"], False, gen, size / 4.6)
    tokens = torch.randint(0, n, (rows,), device="cuda", generator=gen)
    tokens[torch.rand(rows, device="cuda", generator=gen) < 0.1] = -1
    s["tokens"] = tokens
    return s


def run(state):
    if own:
        from rwkv_lightning_cuda_b200 import ops
        if state["op"] == "logprobs":
            names = ("logprobs", "entropy", "lse", "top_ids", "top_logprobs")
            return dict(zip(names, ops.token_logprobs(state["logits"], state["tokens"], top_k=state["top"])))
        if state["op"] == "w4":
            return {"y": ops.linear_w4a16_group(state["x"], state["q"], state["scale"], state["zero"], group_size=state["group"], exact=True)}
        names = ("logprobs", "entropy", "lse")
        return dict(zip(names, ops.head_logprobs(state["x"], state["w"], state["tokens"], scale=state["scale"], zero=state["zero"],
                                                 group_size=state["group"])))
    if state["op"] == "logprobs":
        return _plain_logprobs(state["logits"].float(), state["tokens"], state["top"])
    if state["op"] == "w4":
        return {"y": (state["x"].float() @ _plain_weight4(state).T).half()}
    if state["fmt"] == "f16":
        w = state["w"].float()
    elif state["fmt"] == "w8":
        w = state["w"].float() * state["scale"].float()[:, None]
    else:  # the head's operand is the weight rounded to 16 bits: that is the format's value
        w = _plain_weight4(dict(state, q=state["w"])).half().float()
    got = _plain_logprobs(state["x"].float() @ w.T, state["tokens"][:, None], 0)
    return {"logprobs": got["logprobs"][:, 0], "entropy": got["entropy"], "lse": got["lse"]}


def _plain_weight4(state):
    """The weights that 4-bit codes stand for, in 32 bits: (code - zero) * scale, two codes to a byte, the low one first."""
    q, k = state["q"], state["k"]
    codes = torch.stack((q & 15, q >> 4), dim=2).reshape(q.shape[0], k).float()
    group = torch.arange(k, device=q.device) // state["group"]
    zero = 8.0 if state["zero"] is None else state["zero"].float()[:, group]
    return (codes - zero) * state["scale"].float()[:, group]


def _plain_logprobs(z, tokens, top):
    """Log probabilities of `tokens` [rows, n] under softmax(z), the entropy, the log of the sum of exponentials and the
    `top` likeliest tokens.  A token below 0 asks for nothing (0); a masked one has probability 0; equal ones go by index."""
    rows, vocab = z.shape
    biggest = z.max(dim=1, keepdim=True).values.clamp(min=torch.finfo(torch.float32).min)
    e = (z - biggest).exp()
    total = e.sum(dim=1, keepdim=True)
    empty = total == 0
    log_total = torch.where(empty, torch.zeros_like(total), total.log())
    lse = torch.where(empty, torch.full_like(total, MASKED), biggest + log_total)
    safe = (z - biggest).clamp(min=-1e30)
    entropy = torch.where(empty, torch.zeros_like(total), log_total - (e * safe).sum(dim=1, keepdim=True) / total.clamp(min=1e-30))

    def logprob(ids):
        return (z.gather(1, ids) - biggest) - log_total

    given = torch.where(tokens < 0, torch.zeros((), device=z.device), logprob(tokens.clamp(min=0)))
    out = {"logprobs": given, "entropy": entropy[:, 0], "lse": lse[:, 0], "top_ids": None, "top_logprobs": None}
    if top:
        bits = (z + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -2147483648 - bits, bits)  # the floats' order in whole numbers
        key = order * vocab + (vocab - 1 - torch.arange(vocab, device=z.device))
        ids = key.topk(top, dim=1).indices
        best = logprob(ids)
        out["top_ids"] = torch.where(best == MASKED, torch.full_like(ids, -1), ids).int()
        out["top_logprobs"] = best
    return out


def exact(case, seed):
    s = prepare(case, seed)
    tokens = s.get("tokens")
    if case["op"] == "logprobs":
        parts = []
        for r in range(0, case["rows"], 256):
            parts.append(_exact_logprobs(s["logits"][r:r + 256].double(), tokens[r:r + 256], case["top"]))
        out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
        out["top_ids"] = None
        if not case["top"]:
            out["top_logprobs"] = None
        return out
    x = s["x"].double()
    rows, n, k = case["rows"], case["n"], case["k"]
    y = torch.empty(rows, n, device=x.device, dtype=torch.float64)
    for c in range(0, n, 8192):  # some channels at a time
        w = s["w" if case["op"] == "head" else "q"][c:c + 8192]
        scale = s["scale"][c:c + 8192].double() if s["scale"] is not None else None
        if w.dtype == torch.uint8:
            v = torch.empty(w.shape[0], k, device=x.device, dtype=torch.float64)
            v[:, 0::2] = (w % 16).double()
            v[:, 1::2] = (w // 16).double()
            zero = s["zero"][c:c + 8192].double() if s["zero"] is not None else torch.full_like(scale, 8)
            each = case["group"]
            v -= zero.repeat_interleave(each, dim=1)[:, :k]
            v *= scale.repeat_interleave(each, dim=1)[:, :k]
            if case["op"] == "head":
                v = v.half().double()
        else:
            v = w.double() if scale is None else w.double() * scale[:, None]
        y[:, c:c + 8192] = x @ v.T
    if case["op"] == "w4":
        return {"y": y}
    parts = [_exact_logprobs(y[r:r + 256], tokens[r:r + 256, None], 0) for r in range(0, rows, 256)]
    return {"logprobs": torch.cat([p["logprobs"] for p in parts])[:, 0], "entropy": torch.cat([p["entropy"] for p in parts]),
            "lse": torch.cat([p["lse"] for p in parts])}


def _exact_logprobs(z, tokens, top):
    lse = torch.logsumexp(z, dim=1)
    lp = z - lse[:, None]
    lp[lse == MASKED] = MASKED
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(dim=1)
    rows = torch.arange(z.shape[0], device=z.device)[:, None]
    given = lp[rows, tokens % z.shape[1]]
    given[tokens < 0] = 0
    return {"logprobs": given, "entropy": entropy, "lse": lse, "top_logprobs": lp.sort(dim=1, descending=True).values[:, :max(top, 1)]}
