"""References in 64 bits, and derived tolerances, for the log-probability and group-scaled 4-bit operators."""
import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of fp32
U16 = 2.0 ** -11  # half a step of fp16


def ref_logprobs(z, tokens=None, top=0):
    """Row by row from the definitions: what token_logprobs says about each kind of row."""
    z = z.detach().cpu().double()
    rows, V = z.shape
    n = 0 if tokens is None else tokens.reshape(rows, -1).shape[1]
    lp = torch.zeros(rows, n, dtype=torch.float64)
    H, lse = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    ids = torch.full((rows, top), -1, dtype=torch.int32)
    tlp = torch.full((rows, top), float("-inf"), dtype=torch.float64)
    tok = None if tokens is None else tokens.detach().cpu().reshape(rows, -1)
    for r in range(rows):
        row = z[r]
        if torch.isnan(row).any() or (row == float("inf")).any():
            logp = torch.full((V,), float("nan"), dtype=torch.float64)
            H[r] = lse[r] = float("nan")
            tlp[r] = float("nan")
        elif (row == float("-inf")).all():
            logp = torch.full((V,), float("-inf"), dtype=torch.float64)
            lse[r] = float("-inf")
        else:
            m = row.max()
            total = (row - m).exp().sum()
            logp = (row - m) - total.log()
            lse[r] = m + total.log()
            p = logp.exp()
            H[r] = -(p * logp)[p > 0].sum()
            order = torch.sort(row, descending=True, stable=True).indices[:top]
            order = order[row[order] > float("-inf")]
            ids[r, :len(order)] = order.int()
            tlp[r, :len(order)] = logp[order]
        for i in range(n):
            t = int(tok[r, i])
            lp[r, i] = 0.0 if t < 0 else float("nan") if t >= V else logp[t]
    if tokens is not None:
        lp = lp.reshape(tokens.shape)
    return lp, H, lse, ids, tlp


def softmax_tolerance(V, biggest, logit_error=0.0):
    """How far the log of the sum may be off.  Every term's exponential is off by the rounding of (z - m) log2 e (terms
    with z - m below -30 carry nothing in fp32: 2 * 30 half steps), of exp2 (2 steps) and of the rescaling of partial sums
    (a few more exponentials), 100 half steps in all; the sum of positive terms adds a half step per addition on the longest
    chain (at most V / 512 in a thread, then 64 in the merges), and lse = m + ln s one of itself.  An error of the logits
    enters as it is, once through the sum and once through z."""
    return U32 * (100 + V / 512 + 64 + 2 * abs(biggest)) + 2 * logit_error


def close(got, want, atol, rtol=4 * U32, what=""):
    """Equal NaN and infinities, the rest within atol + rtol |want|."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), what + ": infinities differ"
    fine = torch.isfinite(want)
    off = (got[fine] - want[fine]).abs() - rtol * want[fine].abs()
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= atol, f"{what}: off by {worst:.3g}, allowed {atol:.3g}"


def check_logprobs(got, want, atol, what=""):
    """All five answers of token_logprobs (or three of head_logprobs).  The entropy is ln s - t / s with t / s the mean of
    |z - m| <= ln V + entropy slack: at most 16 for any vocabulary here, each of whose terms is off like the sum's."""
    lp, H, lse = got[:3]
    if lp is not None:
        close(lp, want[0], atol, what=what + " logprobs")
    close(H, want[1], 17 * atol, what=what + " entropy")
    close(lse, want[2], atol, what=what + " lse")
    if len(got) > 3 and got[3] is not None:
        assert torch.equal(got[3].cpu(), want[3]), what + ": alternatives differ"
        close(got[4], want[4], atol, what=what + " top_logprobs")


def w4_weights(q, scale, zero, group, rounded=False, parts=False):
    """(q - zero) * scale in 64 bits, rounded to half where the operator's operand is; `parts`: (q + zero) * scale instead, the size of
    what is added up where codes and zeros are summed apart."""
    q, scale = q.cpu(), scale.cpu().double()
    N, K = q.shape[0], q.shape[1] * 2
    w = torch.stack((q & 15, q >> 4), dim=2).reshape(N, K).double()
    g = torch.arange(K) // group
    z = 8.0 if zero is None else zero.cpu().double()[:, g]
    w = (w + z if parts else w - z) * scale[:, g]
    return w.half().double() if rounded else w


def w4_rounded_any_zero(q, scale, zero, group):
    """The halves that weights count as on the tensor cores when zeros need not be whole numbers: with e the zero as 64 + zero rounded to half
    holds it, half((q - e) scale + half((e - zero) scale)).  Equal to half((q - zero) scale) for whole zeros up to 1024."""
    q, s, z = q.cpu(), scale.cpu().double(), zero.cpu().double()
    N, K = q.shape[0], q.shape[1] * 2
    codes = torch.stack((q & 15, q >> 4), dim=2).reshape(N, K).double()
    held = (64 + z).half().double() - 64
    rest = ((held - z) * s).half().double()
    g = torch.arange(K) // group
    w = (codes - held[:, g]) * s[:, g] + rest[:, g]
    return torch.from_numpy(w.numpy().astype(np.float16)).double()  # (numpy rounds once; torch goes through fp32, which loses a small addend of a tie)


def random_w4(N, K, group, symmetric, gen, device="cuda"):
    q = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=gen)
    groups = -(-K // group)
    scale = ((0.5 + torch.rand(N, groups, generator=gen)) * 0.02).half()
    zero = None if symmetric else torch.randint(0, 16, (N, groups), generator=gen).half()
    return tuple(None if t is None else t.to(device) for t in (q, scale, zero))
