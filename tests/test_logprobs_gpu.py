"""token_logprobs and head_logprobs against 64-bit references, with tolerances derived in tests/head_end.py."""
import pytest
import torch

from tests.head_end import U32, check_logprobs, random_w4, ref_logprobs, softmax_tolerance, w4_weights

pytestmark = pytest.mark.gpu
NEG, POS, NAN = float("-inf"), float("inf"), float("nan")
LOW = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def ops():
    from rwkv_lightning_cuda_b200 import ops as o
    return o


def logits(rows, V, seed=0, half=False, scale=2.5):
    z = torch.randn(rows, V, generator=torch.Generator().manual_seed(seed)) * scale - 4
    return (z.half() if half else z).cuda()


def run_and_check(ops, z, tokens, top, what):
    got = ops.token_logprobs(z, tokens, top_k=top)
    finite = z.float()[torch.isfinite(z.float()) & (z.float() > LOW)]
    biggest = float(finite.abs().max()) if finite.numel() else 0.0
    check_logprobs(got, ref_logprobs(z, tokens, top), softmax_tolerance(z.shape[1], biggest), what)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 2, 5), (3, 31, 32), (2, 257, 0), (5, 4095, 1), (1, 8192, 5), (4, 8193, 32),
                                        (2, 16391, 20), (1, 65536, 20), (3, 70001, 8), (1, 131072, 32), (300, 2049, 4), (75, 20011, 7), (20, 65536, 5)])
def test_shapes(ops, rows, V, top, half):
    z = logits(rows, V, seed=V + rows, half=half)
    tokens = torch.randint(0, V, (rows, 2), generator=torch.Generator().manual_seed(1)).cuda()
    tokens[0, 0] = -1
    tokens[-1, 1] = V
    run_and_check(ops, z, tokens, top, f"{rows}x{V}")


@pytest.mark.parametrize("V", [100, 5000, 65536])
@pytest.mark.parametrize("half", [False, True])
def test_special_rows(ops, V, half):
    """Masks that leave nothing, one or a few tokens, the type's lowest value as a mask, infinities, NaN, ties and sorted rows."""
    z = logits(16, V, seed=7, half=half)
    low = torch.finfo(z.dtype).min
    z[0] = NEG
    z[1] = low
    z[2] = NEG
    z[2, V - 1] = 3
    z[3, 5:] = NEG
    z[4, :V // 2] = low
    z[5, 7] = NAN
    z[6, V - 3] = POS
    z[7] = 1.5
    z[8] = torch.linspace(-5, 5, V).to(z.dtype)
    z[9] = torch.linspace(5, -5, V).to(z.dtype)
    z[10] = (torch.arange(V) % 7).to(z.dtype)
    z[11] = 0
    z[11, ::2] = -0.0
    z[12, 1:] = NAN
    z[13] = POS
    z[14] = NEG
    z[14, 3] = NAN
    z[15] = NEG
    z[15, V // 3:V // 3 + 40] = torch.arange(40).to(z.dtype)
    tokens = torch.stack([torch.zeros(16, dtype=torch.int64), torch.full((16,), V - 1), torch.full((16,), 3)], 1).cuda()
    for top in (0, 1, 20, 32):
        run_and_check(ops, z, tokens, top, f"special V={V} top={top}")


@pytest.mark.parametrize("shift", [0.0, 3000.0, -3000.0])
def test_far_and_peaked_rows(ops, shift):
    z = logits(3, 3001, seed=9, scale=30.0)
    z[0, 17] += 400
    run_and_check(ops, z + shift, torch.tensor([17, 5, 2999]).cuda(), 3, "far")


def strict(ops, z, tokens, top, what):
    """Log probabilities and entropy come from differences to the maximum, so its size adds nothing to what they may be off; lse is held to the
    relative half steps of check_logprobs, which wants NaN where the reference has it and nowhere else.  (30: twice the span of the logits that count.)"""
    got = ops.token_logprobs(z, tokens, top_k=top)
    check_logprobs(got, ref_logprobs(z, tokens, top), softmax_tolerance(z.shape[1], 30.0), what)


@pytest.mark.parametrize("rows,V", [(8, 100), (8, 5000), (8, 65536), (320, 9001)])
@pytest.mark.parametrize("mask", [-1e7, -1e8, -1e9, -1e10, -1e20, -1e30, -1e37, -1e38, LOW])
def test_finite_masks(ops, mask, rows, V):
    """Tokens masked with a large finite number, as samplers and grammars do: most of a row, all of it, the beginning (where a thread sees nothing
    else at first), all but the last, together with -inf; and logits that are themselves of that size."""
    z = logits(rows, V, seed=3)
    gen = torch.Generator().manual_seed(4)
    z[0][(torch.rand(V, generator=gen) < 0.9).cuda()] = mask
    z[1] = mask
    z[2, :V // 2] = mask
    z[3, :V - 1] = mask
    z[4] = mask
    z[4, ::3] = NEG
    z[5, V // 3:] = mask
    z[5, ::2] = NEG
    z[6] = mask
    z[6, 1::2] = mask * 0.5
    if rows > 8:
        z[8:][(torch.rand(rows - 8, V, generator=gen) < 0.9).cuda()] = mask
    tokens = torch.randint(0, V, (rows, 2), generator=gen).cuda()
    for top in (0, 1, 20):
        strict(ops, z, tokens, top, f"mask {mask:g} V={V} top={top}")


@pytest.mark.parametrize("shift", [1e8, -1e8, 1.6e9, -1.6e9, 1e10, -1e10, 1e20, -1e30, 1e38, -2e38])
def test_logits_of_any_size(ops, shift):
    """Rows whose logits are all large: few values a step of fp32 apart, sums of the equal ones.  (At -2e38 the last row holds infinities.)"""
    z = logits(6, 20011, seed=6) + shift
    z[5] = (torch.arange(20011) % 3).cuda() * abs(shift) * 1e-7 + shift
    tokens = torch.randint(0, 20011, (6,), generator=torch.Generator().manual_seed(2)).cuda()
    for top in (0, 5):
        strict(ops, z, tokens, top, f"shift {shift:g} top={top}")


@pytest.mark.parametrize("half", [False, True])
def test_rows_that_start_anywhere(ops, half):
    """Slices: a column offset, a row stride of its own and values behind the rows that must not count."""
    whole = logits(9, 8300, seed=2, half=half)
    whole[:, 0] = 100
    whole[:, 8290:] = POS
    for c in range(1, 6):
        for w in (8200, 8199, 4097, 40):
            z = whole[::2, c:c + w]
            run_and_check(ops, z, torch.full((5,), w - 1).cuda(), 6, f"offset {c} width {w}")


def test_rows_beyond_32_bits(ops):
    """Rows more than 2^31 elements apart."""
    V, ld = 1000, (1 << 30) + 3
    store = torch.empty(2 * ld + V, dtype=torch.float16, device="cuda")
    z = store.as_strided((3, V), (ld, 1))
    z.copy_(logits(3, V, seed=5, half=True))
    run_and_check(ops, z, torch.tensor([1, 2, 3]).cuda(), 4, "far rows")


def test_token_forms_and_absent_outputs(ops):
    z = logits(4, 500)
    lp, H, lse, ids, top = ops.token_logprobs(z)
    assert lp is None and ids is None and top is None and H.shape == (4,) and lse.shape == (4,)
    flat = torch.tensor([1, -1, 499, 10 ** 12]).cuda()
    got = ops.token_logprobs(z, flat)[0]
    assert got.shape == (4,) and float(got[1]) == 0 and bool(torch.isnan(got[3]))
    many = torch.arange(500).cuda().expand(4, 500).contiguous()
    every = ops.token_logprobs(z, many)[0]
    assert float((every.double().exp().sum(1) - 1).abs().max()) < 500 * 4 * U32  # a whole row's probabilities sum to one


def test_one_call_equals_row_by_row(ops):
    """The number of rows chooses how a row is split: answers stay within the tolerance, alternatives are equal; the same call twice is
    equal bit for bit."""
    z = logits(200, 30011, seed=4)
    tok = torch.randint(0, 30011, (200,), generator=torch.Generator().manual_seed(2)).cuda()
    a = ops.token_logprobs(z, tok, top_k=10)
    b = ops.token_logprobs(z, tok, top_k=10)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    for r in (0, 77, 199):
        one = ops.token_logprobs(z[r:r + 1], tok[r:r + 1], top_k=10)
        assert torch.equal(one[3], a[3][r:r + 1])
        for i in (0, 1, 2, 4):
            assert float((one[i] - a[i][r:r + 1]).abs().max()) < 34 * softmax_tolerance(30011, 15)


def test_stream_and_graph_replay(ops):
    """On a side stream, and captured twice: replays answer for what the buffers hold then."""
    z = logits(6, 20000, seed=1)
    tok = torch.randint(0, 20000, (6,), generator=torch.Generator().manual_seed(1)).cuda()
    W = (torch.randn(900, 256, generator=torch.Generator().manual_seed(8)) * 0.05).half().cuda()
    x = torch.randn(6, 256, generator=torch.Generator().manual_seed(9)).half().cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        first = ops.token_logprobs(z, tok, top_k=3)
        h_first = ops.head_logprobs(x, W, tok % 900)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                out = ops.token_logprobs(z, tok, top_k=3) + ops.head_logprobs(x, W, tok % 900)
            graphs.append((g, out))
        for g, out in graphs:
            g.replay()
        for g, out in graphs:
            for u, v in zip(out, first + h_first):
                assert torch.equal(u, v)
        z.mul_(0.5)
        x.mul_(0.5)
        for g, _ in graphs:
            g.replay()
        want = ops.token_logprobs(z, tok, top_k=3) + ops.head_logprobs(x, W, tok % 900)
        for g, out in graphs:
            for u, v in zip(out, want):
                assert torch.equal(u, v)
    st.synchronize()


def test_refusals(ops):
    from rwkv_lightning_cuda_b200 import lib as L
    z, tok = logits(3, 64), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: ops.token_logprobs(z.t()), lambda: ops.token_logprobs(z[:1].expand(3, 64)), lambda: ops.token_logprobs(z, tok[:2]),
                lambda: ops.token_logprobs(z, tok.int()), lambda: ops.token_logprobs(z, tok.cpu()), lambda: ops.token_logprobs(z, top_k=33),
                lambda: ops.token_logprobs(z[:0]), lambda: ops.token_logprobs(z, top_k=2.0), lambda: ops.token_logprobs(z, tok.expand(3, 3).t()[:, :2]),
                lambda: ops.head_logprobs(z.half(), z.half(), tok.int()), lambda: ops.head_logprobs(z.half(), z.half()[:, :32], tok),
                lambda: ops.head_logprobs(z.half()[:, :40].contiguous(), z.half()[:, :40].contiguous(), tok),
                lambda: ops.head_logprobs(z.half(), z.char(), tok), lambda: ops.head_logprobs(z.half().t(), z.half(), tok),
                lambda: ops.head_logprobs(z.half(), z.byte()[:, :32].contiguous(), tok, scale=z.half()[:, :2].contiguous(), group_size=16)):
        with pytest.raises(L.Rwkv7B200Error):
            bad()


# ---- head_logprobs

def head_case(rows, V, K, fmt, group, seed=0, symmetric=False):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=gen).half().cuda()
    tok = torch.randint(0, V, (rows,), generator=gen).cuda()
    tok[rows // 2] = -1
    if fmt == "f16":
        w = (torch.randn(V, K, generator=gen) * 1.3 / K ** 0.5).half().cuda()
        return x, tok, (w, None, None), w.cpu().double()
    if fmt == "w8":
        w = torch.randint(-127, 128, (V, K), dtype=torch.int8, generator=gen).cuda()
        s = (torch.rand(V, generator=gen) * 0.02 / K ** 0.5 + 0.005 / K ** 0.5).half().cuda()
        return x, tok, (w, s, None), w.cpu().double() * s.cpu().double()[:, None]
    q, s, z = random_w4(V, K, group, symmetric, gen)
    s = (s.float() * 10 / K ** 0.5).half()
    return x, tok, (q, s, z), w4_weights(q, s, z, group, rounded=True)


def check_head(ops, x, tok, weight, w64, group, what):
    """A logit is an fp32 sum of K exact products taken 16 (or 32) at a time into one running sum: K / 16 additions, each off by at most
    one step (the tensor cores may truncate) of the largest partial sum, itself at most sum |x w|."""
    w, s, z = weight
    z64 = x.cpu().double() @ w64.T
    error = float((x.cpu().double().abs() @ w64.abs().T).max()) * (x.shape[1] / 16 + 2) * 2 * U32
    got = ops.head_logprobs(x, w, tok, scale=s, zero=z, group_size=group)
    check_logprobs(got, ref_logprobs(z64, tok), softmax_tolerance(w64.shape[0], float(z64.abs().max()), error), what)


@pytest.mark.parametrize("fmt,group,symmetric", [("f16", 128, False), ("w8", 128, False), ("w4", 32, False), ("w4", 64, True), ("w4", 128, False)])
@pytest.mark.parametrize("rows,V,K", [(1, 1, 32), (2, 100, 64), (3, 257, 96), (17, 1000, 160), (77, 515, 768), (129, 2001, 416), (300, 256, 256), (5, 40000, 128),
                                      (640, 4100, 288)])
def test_head_shapes(ops, rows, V, K, fmt, group, symmetric):
    x, tok, weight, w64 = head_case(rows, V, K, fmt, group, seed=rows + V + K, symmetric=symmetric)
    check_head(ops, x, tok, weight, w64, group, f"{fmt} {rows}x{V}x{K}")


@pytest.mark.parametrize("fmt,group", [("f16", 128), ("w8", 128), ("w4", 32), ("w4", 64), ("w4", 128)])
@pytest.mark.parametrize("rows,V,K", [(9, 300, 2080), (70, 129, 4128), (130, 515, 8192), (300, 200, 3136)])
def test_head_long_k(ops, rows, V, K, fmt, group):
    """Long sums go in ranges: tiles and blocks of their own, tails of a range and of a stage."""
    check_head(ops, *head_case(rows, V, K, fmt, group, seed=K), group, f"{rows}x{V}x{K} {fmt} g{group}")


@pytest.mark.parametrize("fmt,group", [("f16", 128), ("w8", 128), ("w4", 32), ("w4", 128)])
@pytest.mark.parametrize("rows", [9, 64, 300])
@pytest.mark.parametrize("K", [4096, 8192])
def test_head_long_k_loses_no_more_than_a_range(ops, K, rows, fmt, group):
    """What the tensor cores cut off of what they add to a running sum stays that of 1024 products, however long K is: 64 additions, each off by half a
    step (2^-23) on average, of a partial sum that averages half of the whole, 64 / 4 * 2^-23 = 1.9e-6 of a logit's size, root mean square.  (Measured 0.9e-6 to
    1.4e-6; with all of K in one sum 4.3e-6 to 5.0e-6 at 4096 and 8e-6 to 10e-6 at 8192.)  Logits of about 100, so that the answers' own
    rounding to fp32 does not count."""
    gen = torch.Generator(device="cuda").manual_seed(K + rows)
    V, s, z = 3000, None, None
    x = torch.randn(rows, K, device="cuda", generator=gen).half()
    if fmt == "f16":
        w = (torch.randn(V, K, device="cuda", generator=gen) * (100 / K ** 0.5)).half()
        w64 = w.double()
    elif fmt == "w8":
        w = torch.randint(-127, 128, (V, K), device="cuda", generator=gen, dtype=torch.int8)
        s = ((0.5 + torch.rand(V, device="cuda", generator=gen)) * (100 / 74 / K ** 0.5)).half()
        w64 = w.double() * s.double()[:, None]
    else:
        w = torch.randint(0, 256, (V, K // 2), device="cuda", generator=gen, dtype=torch.uint8)
        s = ((0.5 + torch.rand(V, K // group, device="cuda", generator=gen)) * (100 / 4.6 / K ** 0.5)).half()
        z = torch.randint(4, 12, (V, K // group), device="cuda", generator=gen).half()
        w64 = w4_weights(w, s, z, group, rounded=True).cuda()
    z64 = x.double() @ w64.T
    off, size = [], []
    for _ in range(4):
        tok = torch.randint(0, V, (rows,), device="cuda", generator=gen)
        lp, _, lse = ops.head_logprobs(x, w, tok, scale=s, zero=z, group_size=group)
        size.append(z64.gather(1, tok[:, None])[:, 0])
        off.append(lp.double() + lse.double() - size[-1])  # the given token's logit
    assert float(torch.cat(off).norm() / torch.cat(size).norm()) <= 64 / 4 * 2.0 ** -23


def test_head_special_rows(ops):
    """A row whose logits overflow answers NaN and leaves its neighbours alone; ids outside the vocabulary; no tokens at all."""
    x, tok, (w, _, _), w64 = head_case(6, 300, 64, "f16", 128)
    x[2, 5] = POS
    x[4] = NAN
    tok[0], tok[1] = 300, 10 ** 11
    z = x.cpu().double() @ w64.T
    got = ops.head_logprobs(x, w, tok)
    fine = [0, 1, 3, 5]
    want = ref_logprobs(z, tok)
    check_logprobs([g[fine] for g in got], [v[fine] for v in want[:3]], softmax_tolerance(300, 8, 1e-4), "neighbours")
    assert bool(torch.isnan(got[1][[2, 4]]).all()) and bool(torch.isnan(got[2][[2, 4]]).all())
    none = ops.head_logprobs(x, w)
    assert none[0] is None and torch.equal(none[1][fine], got[1][fine])


def test_head_equals_product_then_logprobs(ops):
    """The two routes to a prompt's log probabilities: the fused product, and logits (rounded to half) followed by token_logprobs."""
    from rwkv_lightning_cuda_b200 import lib as L
    x, tok, (w, _, _), w64 = head_case(40, 3000, 512, "f16", 128, seed=3)
    z = ops.linear_f16_orig(x, w, epilogue=L.EPI_F32)
    two = ops.token_logprobs(z, tok)
    one = ops.head_logprobs(x, w, tok)
    biggest = float(z.abs().max())
    assert float((one[0] - two[0]).abs().max()) <= 2 * biggest * 2 ** -11 + 1e-4  # both the given logit and the sum move by a half step of fp16
    assert float((one[2] - two[2]).abs().max()) <= biggest * 2 ** -11 + 1e-4


@pytest.mark.parametrize("V,K", [(65536, 1024), (70001, 1024), (65536, 1056), (33000, 2080), (16411, 4096), (4099, 16384), (8200, 16416)])
def test_head_one_row_of_a_large_matrix(ops, V, K):
    """The form of a scored decode step: one row on an fp16 head of 128 MB and more, which streams the weights (up to K = 16384) and keeps its
    logits for a second pass; the given token, none given, ids outside, and the same call again."""
    gen = torch.Generator(device="cuda").manual_seed(V + K)
    w = torch.empty(V, K, dtype=torch.float16, device="cuda").normal_(0, 1.3 / K ** 0.5, generator=gen)
    x = torch.randn(1, K, device="cuda", generator=gen).half()
    z64, size = torch.empty(1, V, dtype=torch.float64), 0.0
    for c in range(0, V, 8192):
        part = w[c:c + 8192].double()
        z64[:, c:c + 8192] = (x.double() @ part.T).cpu()
        size = max(size, float((x.double().abs() @ part.abs().T).max()))
        del part
    tol = softmax_tolerance(V, float(z64.abs().max()), size * (K / 16 + 2) * 2 * U32)  # as check_head
    for token in (0, V - 1, V // 3, -1, V):
        tok = torch.tensor([token]).cuda()
        got = ops.head_logprobs(x, w, tok)
        check_logprobs(got, ref_logprobs(z64, tok), tol, f"{V}x{K} token {token}")
        for a, b in zip(got, ops.head_logprobs(x, w, tok)):
            assert torch.equal(a, b) or bool(torch.isnan(a).all() and torch.isnan(b).all())
    none = ops.head_logprobs(x, w)
    assert none[0] is None and torch.equal(none[1], got[1]) and torch.equal(none[2], got[2])
    two = ops.head_logprobs(x.expand(2, K).contiguous(), w)  # (the other route)
    assert float((two[2] - none[2]).abs().max()) <= 2 * tol


def test_head_weights_made_just_before(ops):
    """One row on a large fp16 matrix that the kernel before it on the stream writes, itself one that lets its successor begin early: the answer is that
    of the finished weights, every time."""
    gen = torch.Generator().manual_seed(21)
    V, K = 65536, 1024
    q, s, _ = random_w4(K, 32, 32, True, gen)
    made = [torch.randn(V, 32, generator=gen).half().cuda() for _ in range(2)]
    x, tok = torch.randn(1, K, generator=gen).half().cuda(), torch.tensor([V - 1]).cuda()
    first = []
    for m in made:
        w = ops.linear_w4a16_group(m, q, s, None, 32)
        torch.cuda.synchronize()
        first.append(ops.head_logprobs(x, w, tok))
        del w
    for i in range(12):
        w = ops.linear_w4a16_group(made[i % 2], q, s, None, 32)
        got = ops.head_logprobs(x, w, tok)
        for a, b in zip(got, first[i % 2]):
            assert torch.equal(a, b)
        del w, got
