"""4-bit weights with group scales: packing, the product and the whole head end, against 64-bit references."""
import numpy as np
import pytest
import torch

from tests.head_end import U16, U32, check_logprobs, random_w4, ref_logprobs, softmax_tolerance, w4_rounded_any_zero, w4_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rwkv_lightning_cuda_b200 import ops as o
    return o


def check_product(y, x, weight, group, what):
    """fp32 sums of K products: at most K / 16 additions to one running sum and 64 more in the merges, each off by at most one step of what has
    been added up, codes and zeros apart: sum |x| (q + zero) scale.  Then one rounding to half (half a step, or of the smallest subnormal).
    Beyond 8 rows the weights are rounded to half first."""
    x64 = x.cpu().double()
    want = x64 @ w4_weights(*weight, group, rounded=x.shape[0] > 8).T
    size = x64.abs() @ w4_weights(*weight, group, parts=True).T
    bound = size * (x.shape[1] / 16 + 64) * 2 * U32 + want.abs() * U16 * (1 + 1e-3) + 2.0 ** -25
    got = y.detach().cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs() - bound
    assert float(off.max()) <= 0, f"{what}: off by {float((got - want).abs().max()):.3g}"


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 32), (5, 96), (16, 256), (33, 1056)])
def test_pack_and_unpack(ops, N, K, group, symmetric):
    """Scales, zeros and codes from the formulas in numpy's fp32, bit for bit; unpacking gives the codes' values rounded once."""
    rng = np.random.default_rng(N + K + group)
    W = (rng.standard_normal((N, K)) * 0.05).astype(np.float16)
    W[0, :32] = 0
    q, s, z = ops.quant_pack_w4_group(torch.from_numpy(W).cuda(), group, symmetric)
    G = -(-K // group)
    f = np.float32
    for n in range(N):
        for g in range(G):
            w = W[n, g * group:(g + 1) * group].astype(f)
            mn, mx = min(f(0), w.min()), max(f(0), w.max())
            sc = np.float16(max(-mn, mx) / f(7)) if symmetric else np.float16((mx - mn) / f(15))
            zero = f(8) if symmetric else f(0)
            if not symmetric and sc > 0:
                zero = f(np.clip(np.rint(-mn / f(sc)), 0, 15))
            codes = np.clip(np.rint(w / f(sc)) + zero, 0, 15) if sc > 0 else np.full_like(w, zero)
            assert float(s[n, g]) == float(sc) and (symmetric or float(z[n, g]) == float(zero))
            row = q[n].cpu().numpy()[g * group // 2:(g * group + len(w)) // 2]
            assert ((row & 15) == codes[0::2]).all() and ((row >> 4) == codes[1::2]).all()
    back = ops.quant_unpack_w4_group(q, s, z, group).cpu().double()
    assert torch.equal(back, w4_weights(q, s, z, group, rounded=True))


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 7, 64), (1, 300, 2080), (2, 64, 256), (3, 130, 512), (4, 2561, 1056), (5, 20, 4096), (8, 1000, 416),
                                   (9, 33, 288), (16, 65, 2048), (1, 40, 16384), (7, 24, 16416), (16, 48, 10272)])
def test_few_rows(ops, M, N, K, group, symmetric):
    gen = torch.Generator().manual_seed(M + N + K + group)
    q, s, z = random_w4(N, K, group, symmetric, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    check_product(ops.linear_w4a16_group(x, q, s, z, group), x, (q, s, z), group, f"{M}x{N}x{K} g{group}")


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(17, 128, 128), (33, 130, 416), (96, 1024, 2560), (200, 37, 1056), (256, 516, 288), (300, 40, 4128), (513, 4, 96)])
def test_many_rows(ops, M, N, K, group, symmetric):
    gen = torch.Generator().manual_seed(M + N + K + group)
    q, s, z = random_w4(N, K, group, symmetric, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    check_product(ops.linear_w4a16_group(x, q, s, z, group), x, (q, s, z), group, f"{M}x{N}x{K} g{group}")


def check_exact(y, x, weight, group, what):
    """As check_product at any number of rows: no weight is rounded.  With 9 rows and more a weight is two halves, whose products come one after the
    other: K / 8 additions to the running sum instead of K / 16."""
    x64 = x.cpu().double()
    want = x64 @ w4_weights(*weight, group).T
    size = x64.abs() @ w4_weights(*weight, group, parts=True).T
    bound = size * (x.shape[1] / 8 + 64) * 2 * U32 + want.abs() * U16 * (1 + 1e-3) + 2.0 ** -25
    off = (y.detach().cpu().double() - want).abs() - bound
    assert float(off.max()) <= 0, f"{what}: off by {float((y.cpu().double() - want).abs().max()):.3g}"


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 40, 288), (8, 33, 96), (9, 33, 288), (16, 65, 32), (17, 128, 128), (33, 130, 416), (65, 300, 64), (96, 1024, 2560), (129, 128, 160),
                                   (200, 37, 1056), (256, 516, 288), (300, 40, 4128), (513, 4, 96)])
def test_exact_products(ops, M, N, K, group, symmetric):
    """Asked for, no weight is rounded with many rows either: at short K the rounding of the weights is several times what this allows."""
    gen = torch.Generator().manual_seed(M + N + K + group)
    q, s, z = random_w4(N, K, group, symmetric, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    check_exact(ops.linear_w4a16_group(x, q, s, z, group, exact=True), x, (q, s, z), group, f"{M}x{N}x{K} g{group}")


def test_exact_products_one_weight_at_a_time(ops):
    """Every code, zero and place of a word against one activation: the weight itself, rounded once to half, at scales that need all their bits."""
    K, N, group = 256, 256, 32
    for code in range(16):
        w = torch.full((N, K), 5, dtype=torch.uint8)
        w[torch.arange(N), torch.arange(K)] = code
        q = (w[:, 0::2] | (w[:, 1::2] << 4)).cuda()
        s = (1 + torch.arange(1, N * K // group + 1).reshape(N, -1) / 1024 * 0.999).half().cuda()
        z = (torch.arange(N * K // group).reshape(N, -1) % 16).half().cuda()
        x = torch.eye(K).half().cuda()  # row m picks weight m of every channel
        y = ops.linear_w4a16_group(x, q, s, z, group, exact=True)
        want = w4_weights(q, s, z, group).T
        assert torch.equal(y.cpu(), want.half())
        assert torch.equal(ops.linear_w4a16_group(torch.cat([x, -x]), q, s, z, group, exact=True)[K:], -y)


def test_exact_products_keep_what_rounding_takes_off(ops):
    """Activations of opposite sign on two weights whose difference is not a whole number of the steps they would be rounded to: it survives."""
    M, N, K, group = 40, 64, 64, 32
    w = torch.zeros(N, K, dtype=torch.uint8)
    w[:, 0], w[:, 32] = 15, 15
    q = (w[:, 0::2] | (w[:, 1::2] << 4)).cuda()
    base = 1 + torch.arange(N) / 1024
    s = torch.stack([base, base + 1 / 1024], 1).half().cuda()  # 15 * 2^-10 apart, weights with steps of 2^-7
    z = torch.zeros(N, 2).half().cuda()
    x = torch.zeros(M, K).half().cuda()
    x[:, 0], x[:, 32] = -1, 1
    want = (15 * (s[:, 1].double() - s[:, 0].double())).half()
    assert torch.equal(ops.linear_w4a16_group(x, q, s, z, group, exact=True), want.expand(M, N))


def test_exact_epilogues_and_repeats(ops):
    from rwkv_lightning_cuda_b200 import lib as L
    gen = torch.Generator().manual_seed(12)
    q, s, z = random_w4(516, 2080, 32, False, gen)
    for M in (5, 9, 20, 70, 150, 260):
        x = torch.randn(M, 2080, generator=gen).half().cuda()
        y = ops.linear_w4a16_group(x, q, s, z, 32, exact=True)
        y32 = ops.linear_w4a16_group(x, q, s, z, 32, epilogue=L.EPI_F32, exact=True)
        assert y32.dtype == torch.float32 and torch.equal(y32, y.float())
        relu2 = ops.linear_w4a16_group(x, q, s, z, 32, epilogue=L.EPI_RELU2, exact=True)
        assert torch.equal(relu2, (y.float().clamp(min=0) ** 2).half())
        for _ in range(10):
            assert torch.equal(ops.linear_w4a16_group(x, q, s, z, 32, exact=True), y)


def test_epilogues(ops):
    from rwkv_lightning_cuda_b200 import lib as L
    gen = torch.Generator().manual_seed(2)
    q, s, z = random_w4(70, 320, 64, False, gen)
    for M in (1, 6, 20, 70):
        x = torch.randn(M, 320, generator=gen).half().cuda()
        y = ops.linear_w4a16_group(x, q, s, z, 64)
        y32 = ops.linear_w4a16_group(x, q, s, z, 64, epilogue=L.EPI_F32)
        assert y32.dtype == torch.float32 and torch.equal(y32, y.float())
        relu2 = ops.linear_w4a16_group(x, q, s, z, 64, epilogue=L.EPI_RELU2)
        assert torch.equal(relu2, (y.float().clamp(min=0) ** 2).half())


@pytest.mark.parametrize("M", [1, 3, 8, 40])
def test_small_and_special_activations(ops, M):
    """Activations down to the smallest subnormal half keep their value, large ones do not overflow in between, and an infinity or NaN stays in
    its row."""
    gen = torch.Generator().manual_seed(5)
    q, s, z = random_w4(48, 512, 64, False, gen)
    x = (torch.randn(M, 512, generator=gen) * 2e-6).half().cuda()
    wide = (s.float() * 50).half()
    check_product(ops.linear_w4a16_group(x, q, wide, z, 64), x, (q, wide, z), 64, "subnormal activations")
    big = (torch.randn(M, 512, generator=gen) * 2000).half().cuda()
    check_product(ops.linear_w4a16_group(big, q, s, z, 64), big, (q, s, z), 64, "large activations")
    if M > 1:
        x = torch.randn(M, 512, generator=gen).half().cuda()
        clean = ops.linear_w4a16_group(x, q, s, z, 64)
        x[1, 100] = float("nan")
        got = ops.linear_w4a16_group(x, q, s, z, 64)
        keep = [m for m in range(M) if m != 1]
        assert torch.equal(got[keep], clean[keep]) and bool(torch.isnan(got[1]).all())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K", [32, 96, 288, 544])
def test_nothing_behind_k_counts(ops, K, group):
    """Scales at which code 0 would be an infinite half, but no code that is there: the places behind K, which read as code 0, add nothing."""
    gen = torch.Generator().manual_seed(K + group)
    N = 70
    w = torch.randint(8, 12, (N, K), generator=gen, dtype=torch.uint8)
    q = (w[:, 0::2] | (w[:, 1::2] << 4)).cuda()
    s = torch.full((N, -(-K // group)), 16384.0).half().cuda()
    for M in (1, 8, 20):
        x = (torch.randn(M, K, generator=gen) * 1e-4).half().cuda()
        check_product(ops.linear_w4a16_group(x, q, s, None, group), x, (q, s, None), group, f"{M} rows of {K}")
        want = torch.log_softmax(x.cpu().double() @ w4_weights(q, s, None, group, rounded=True).T, dim=1)
        tok = torch.randint(0, N, (M,), generator=gen)
        lp, entropy, lse = ops.head_logprobs(x, q, tok.cuda(), scale=s, group_size=group)
        # logits: as in check_product without the rounding to half; log probabilities twice that and some steps of their own
        size = (x.cpu().double().abs() @ w4_weights(q, s, None, group, parts=True).T).max()
        tol = 2 * float(size) * (K / 16 + 64) * 2 * U32 + 200 * U32 * (1 + float(want.abs().max()))
        assert float((lp.cpu().double() - want[torch.arange(M), tok]).abs().max()) <= tol
        assert bool(torch.isfinite(entropy).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("M,N,K", [(100, 200, 6176), (128, 200, 3136), (200, 2000, 6176)])
def test_long_products_again_and_again(ops, M, N, K):
    """Rings that go round many times under slow expansion (two groups to 64 weights): the same right answer every time."""
    gen = torch.Generator().manual_seed(K)
    q, s, z = random_w4(N, K, 32, False, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    first = ops.linear_w4a16_group(x, q, s, z, 32)
    check_product(first, x, (q, s, z), 32, "first")
    for _ in range(30):
        assert torch.equal(ops.linear_w4a16_group(x, q, s, z, 32), first)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 24, 57344), (1, 24, 65536), (3, 130, 70016), (8, 7, 98304), (9, 7, 98304)])
def test_few_rows_of_a_long_k(ops, M, N, K, group):
    """Rows that do not fit into shared memory go another way, with weights that are not rounded either."""
    gen = torch.Generator().manual_seed(M + K)
    q, s, z = random_w4(N, K, group, False, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    check_exact(ops.linear_w4a16_group(x, q, s, z, group, exact=M > 8), x, (q, s, z), group, f"{M}x{N}x{K} g{group}")


@pytest.mark.parametrize("M,N,K", [(1, 8192, 65536), (9, 1024, 32768), (100, 512, 65536), (300, 256, 24576)])
def test_exact_products_of_a_long_k_lose_no_more_than_a_range(ops, M, N, K):
    """What the tensor cores cut off is a bias towards zero, which the mean over many results shows below their rounding to half: at most that of
    8192 products, twice 512 additions, each off by half a step (2^-23) on average of a sum that averages half of the whole, 1024 / 4 * 2^-23."""
    gen = torch.Generator(device="cuda").manual_seed(K + M)
    q = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device="cuda", generator=gen)
    s = ((0.5 + torch.rand(N, K // 64, device="cuda", generator=gen)) * 0.02).half()
    z = torch.randint(4, 12, (N, K // 64), device="cuda", generator=gen).half()
    x = torch.randn(M, K, device="cuda", generator=gen).half()
    y = ops.linear_w4a16_group(x, q, s, z, 64, exact=True).double()
    want = x.double() @ w4_weights(q, s, z, 64).cuda().T
    bias = float(((y - want) * want.sign()).sum() / want.abs().sum())
    noise = 5 * float((want.abs() * U16).norm() / want.abs().sum())  # of the results' own rounding
    assert abs(bias) <= 1024 / 4 * 2.0 ** -23 + noise, bias


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("off", [1, 2, 5])
def test_scales_and_zeros_that_start_anywhere(ops, off, group):
    """Parameters that begin off a 16-byte or 4-byte boundary, as slices of a file's buffer do: the answers of aligned ones."""
    gen = torch.Generator().manual_seed(off + group)
    N, K = 300, 2048
    q, s, z = random_w4(N, K, group, False, gen)
    z = (z + 0.25 * torch.randint(0, 2, z.shape, generator=gen).cuda()).half()

    def moved(t):
        store = torch.full((t.numel() + off,), float("nan"), dtype=torch.float16, device="cuda")
        store[off:] = t.flatten()
        return store[off:].view(t.shape)
    for M in (1, 3, 8, 9, 70, 200):
        x, tok = torch.randn(M, K, generator=gen).half().cuda(), torch.randint(0, N, (M,), generator=gen).cuda()
        for zero in (z, None):
            there = None if zero is None else moved(zero)
            for exact in (False, True):
                y = ops.linear_w4a16_group(x, q, moved(s), there, group, exact=exact)
                assert torch.equal(y, ops.linear_w4a16_group(x, q, s, zero, group, exact=exact)), f"{M} rows, exact={exact}"
            got, want = ops.head_logprobs(x, q, tok, scale=moved(s), zero=there, group_size=group), ops.head_logprobs(x, q, tok, scale=s, zero=zero, group_size=group)
            assert all(torch.equal(u, v) for u, v in zip(got, want)), f"head, {M} rows"


def fractional_w4(N, K, group, gen, which):
    """Zeros between whole numbers: everywhere, in one channel of forty, or in one group.  (For up to eight rows of the head from 2 on, so that
    (q - zero) * scale has 24 bits at most and the 64-bit reference's single rounding to half is that of a product in fp32.)"""
    q, s, z = random_w4(N, K, group, False, gen)
    f = (2 + 13.99 * torch.rand(z.shape, generator=gen)).half().cuda()
    if which == "channels":
        z[::40] = f[::40]
    elif which == "group":
        z[:, z.shape[1] // 2] = f[:, z.shape[1] // 2]
    else:
        z = f
    return q, s, z


@pytest.mark.parametrize("which", ["all", "channels", "group"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 70, 288), (5, 33, 2080), (8, 200, 1024), (9, 33, 288), (17, 300, 1024), (33, 130, 416), (100, 516, 2048), (200, 200, 1056), (300, 130, 512)])
def test_zeros_that_are_not_whole(ops, M, N, K, group, which):
    """fp16 zeros as common formats have them: in products at any number of rows, and in the head, whose weights are halves."""
    gen = torch.Generator().manual_seed(M + N + K + group)
    q, s, z = fractional_w4(N, K, group, gen, which)
    x = torch.randn(M, K, generator=gen).half().cuda()
    x64, size = x.cpu().double(), x.cpu().double().abs() @ w4_weights(q, s, z, group, parts=True).T
    halves = w4_weights(q, s, z, group, rounded=True) if M <= 8 else w4_rounded_any_zero(q, s, z, group)
    # products: the bound of check_product; exact with nine rows and more: check_exact's, and 1.5 * 2^-16 of the scale (the rounding of what the zero
    # leaves over, times the scale, a 32nd of it: 2^-17; and of the low half that it is added to, below a 16th: 2^-16) and the smallest half's per weight
    y = ops.linear_w4a16_group(x, q, s, z, group).cpu().double()
    want = x64 @ (w4_weights(q, s, z, group) if M <= 8 else halves).T
    assert float(((y - want).abs() - size * (K / 16 + 64) * 2 * U32 - want.abs() * U16 * (1 + 1e-3) - 2.0 ** -25).max()) <= 0
    y = ops.linear_w4a16_group(x, q, s, z, group, exact=True).cpu().double()
    want = x64 @ w4_weights(q, s, z, group).T
    slack = x64.abs() @ (1.5 * 2.0 ** -16 * s.cpu().double()[:, torch.arange(K) // group] + 2.0 ** -25).T
    assert float(((y - want).abs() - size * (K / 8 + 64) * 2 * U32 - slack - want.abs() * U16 * (1 + 1e-3) - 2.0 ** -25).max()) <= 0
    tok = torch.randint(0, N, (M,), generator=gen).cuda()
    z64 = x64 @ halves.T
    error = float((x64.abs() @ halves.abs().T).max()) * (K / 16 + 2) * 2 * U32  # as for every head: K / 16 additions to one running sum
    got = ops.head_logprobs(x, q, tok, scale=s, zero=z, group_size=group)
    check_logprobs(got, ref_logprobs(z64, tok), softmax_tolerance(N, float(z64.abs().max()), error), f"head {M}x{N}x{K} g{group}")


def test_small_and_odd_zeros_one_weight_at_a_time(ops):
    """Every code against zeros below 2, below 0 and far from the codes, weight by weight.  What 64 + zero leaves over is at most half a step of it,
    2^-12 (64 + |zero|), times the scale: rounded once in a weight that is a half, and with the low half once more in one that is two."""
    K, N, group = 128, 128, 32
    zeros = torch.tensor([0.0, 0.1, 0.3337, 1.7, 1.999, -0.25, -3.3, 15.99, 16.5, 100.0, 100.3, 1023.0, 6e-8, -100.0, 7.5, 8.0]).half()
    w = torch.arange(K)[None].add(torch.arange(N)[:, None]).remainder(16).to(torch.uint8)
    q = (w[:, 0::2] | (w[:, 1::2] << 4)).cuda()
    s = (1 + torch.arange(N * 4).reshape(N, 4) / 1024).half().cuda()
    z = zeros[torch.arange(N * 4).reshape(N, 4).remainder(16)].cuda()
    x = torch.eye(K).half().cuda()
    want = w4_weights(q, s, z, group).T
    g = torch.arange(K) // group
    s64, z64 = s.cpu().double()[:, g].T, z.cpu().double()[:, g].T
    left = 2.0 ** -12 * (64 + z64.abs()) * s64
    for M in (8, 40, 128):
        y = ops.linear_w4a16_group(x[:M], q, s, z, group, exact=True).cpu().double()
        # (up to eight rows codes and zeros are summed apart in fp32: a few half steps of the larger one)
        slack = 4 * U32 * ((15 + z64.abs()) * s64)[:M] if M <= 8 else 3 * U16 * left[:M] + 2.0 ** -25
        assert float(((y - want[:M]).abs() - want[:M].abs() * U16 * (1 + 1e-3) - slack - 2.0 ** -25).max()) <= 0
    halves = w4_rounded_any_zero(q, s, z, group).T
    assert float(((halves - want).abs() - want.abs() * U16 * (1 + 1e-3) - U16 * left - 2.0 ** -25).max()) <= 0
    for M in (40, 128):
        assert torch.equal(ops.linear_w4a16_group(x[:M], q, s, z, group).cpu().double(), halves[:M])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 8192), (1, 20000, 2080), (2, 5000, 4096), (3, 2561, 6176), (5, 9000, 3136), (8, 4000, 8192)])
def test_streamed_products_again_and_again(ops, M, N, K, group):
    """Few rows, whose rings are refilled behind the products: the right answer, and the same one every time; the head's form of them too."""
    gen = torch.Generator().manual_seed(K + M)
    q, s, z = random_w4(N, K, group, False, gen)
    x = torch.randn(M, K, generator=gen).half().cuda()
    tok = torch.randint(0, N, (M,), generator=gen).cuda()
    first, scores = ops.linear_w4a16_group(x, q, s, z, group), ops.head_logprobs(x, q, tok, scale=s, zero=z, group_size=group)
    check_product(first, x, (q, s, z), group, "first")
    got = [(ops.linear_w4a16_group(x, q, s, z, group), ops.head_logprobs(x, q, tok, scale=s, zero=z, group_size=group)) for _ in range(40)]
    for y, l in got:
        assert torch.equal(y, first) and all(torch.equal(u, v) for u, v in zip(l, scores))


def test_codes_one_at_a_time(ops):
    """Each of the 16 codes at each place of a word, and each group's own scale: one weight at a time against one activation."""
    K, group = 288, 32
    for code in range(16):
        N = K
        w = torch.full((N, K), 3, dtype=torch.uint8)
        w[torch.arange(K), torch.arange(K)] = code
        q = (w[:, 0::2] | (w[:, 1::2] << 4)).cuda()
        s = torch.linspace(0.5, 2, K // group).half().expand(N, -1).contiguous().cuda()
        z = torch.full((N, K // group), 3.0).half().cuda()
        x = torch.arange(1, K + 1).half()[None].cuda()
        y = ops.linear_w4a16_group(x, q, s, z, group)
        want = (code - 3) * torch.arange(1, K + 1).double() * s[0].cpu().double().repeat_interleave(group)
        assert torch.equal(y[0].cpu(), want.half())


def test_two_calls_and_replays_are_equal(ops):
    gen = torch.Generator().manual_seed(6)
    q, s, z = random_w4(515, 2080, 128, False, gen)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for M in (1, 5, 24, 100):
            x = torch.randn(M, 2080, generator=gen).half().cuda()
            a, b = ops.linear_w4a16_group(x, q, s, z, 128), ops.linear_w4a16_group(x, q, s, z, 128)
            assert torch.equal(a, b)
            graphs = []
            for _ in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    graphs.append((ops.linear_w4a16_group(x, q, s, z, 128), g))
            x.mul_(0.5)
            for _, g in graphs:
                g.replay()
            want = ops.linear_w4a16_group(x, q, s, z, 128)
            for y, _ in graphs:
                assert torch.equal(y, want)
    st.synchronize()


def test_refusals(ops):
    from rwkv_lightning_cuda_b200 import lib as L
    q, s, z = random_w4(8, 128, 64, False, torch.Generator().manual_seed(1))
    x = torch.zeros(2, 128, dtype=torch.float16, device="cuda")
    for bad in (lambda: ops.linear_w4a16_group(x, q, s, z, 32), lambda: ops.linear_w4a16_group(x, q, s, z[:, :1].contiguous(), 64),
                lambda: ops.linear_w4a16_group(x.float(), q, s, z, 64), lambda: ops.linear_w4a16_group(x[:, :64], q, s, z, 64),
                lambda: ops.linear_w4a16_group(x, q.t(), s, z, 64), lambda: ops.linear_w4a16_group(x[:0], q, s, z, 64),
                lambda: ops.linear_w4a16_group(x, q, s.float(), z, 64), lambda: ops.linear_w4a16_group(x, q, s, z, 64, epilogue=2),
                lambda: ops.linear_w4a16_group(x.cpu(), q, s, z, 64), lambda: ops.quant_pack_w4_group(x[:, :40].contiguous(), 32),
                lambda: ops.quant_unpack_w4_group(q, s, z, 128)):
        with pytest.raises(L.Rwkv7B200Error):
            bad()


def test_head_end_of_a_step(ops):
    """The run a decode step ends with: a 4-bit head in fine groups, logits in fp32, then the chosen token's log probability with alternatives; and the
    fused route over the same weights."""
    from rwkv_lightning_cuda_b200 import lib as L
    gen = torch.Generator().manual_seed(11)
    W = (torch.randn(5003, 256, generator=gen) * 0.08).half().cuda()
    x = torch.randn(3, 256, generator=gen).half().cuda()
    q, s, z = ops.quant_pack_w4_group(W, 32)
    logits = ops.linear_w4a16_group(x, q, s, z, 32, epilogue=L.EPI_F32)
    chosen = ops.greedy_pick(logits)
    got = ops.token_logprobs(logits, chosen.long(), top_k=5)
    check_logprobs(got, ref_logprobs(logits, chosen.long(), 5), softmax_tolerance(5003, float(logits.abs().max())), "step")
    assert torch.equal(got[3][:, 0], chosen) and torch.equal(got[4][:, 0], got[0])
    fused = ops.head_logprobs(x, q, chosen.long(), scale=s, zero=z, group_size=32)
    # the logits of the first route are rounded to half, the weights of the second
    size = float((x.double().abs() @ w4_weights(q, s, z, 32).abs().T.cuda()).max())
    slack = 2 * (float(logits.abs().max()) * U16 + size * U16) + softmax_tolerance(5003, 10)
    assert float((fused[0] - got[0]).abs().max()) <= slack
