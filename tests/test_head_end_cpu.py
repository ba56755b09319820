"""Refusals of the log-probability and group-scaled 4-bit entry points: status codes before anything is enqueued, and the
Python layer's checks.  No GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from rwkv_lightning_cuda_b200 import build, lib as L
    build.build()
    return L.load_library()


P = C.c_void_p(1 << 20)  # an aligned address that nothing reads: every call below is refused first


def test_token_logprobs_refusals(lib):
    def call(rows=1, V=8, logits=P, dtype=2, ld=8, tokens=P, n=1, top=1, lp=P, ids=P, top_lp=P):
        return lib.rwkv7_b200_token_logprobs(None, rows, V, logits, dtype, ld, tokens, n, top, lp, None, None, ids, top_lp)
    assert call(rows=0) == 1 and call(V=0) == 1 and call(logits=None) == 1 and call(rows=-3) == 1
    assert call(dtype=1) == 1 and b"dtype" in lib.rwkv7_b200_last_error()
    assert call(ld=7) == 2 and b"stride" in lib.rwkv7_b200_last_error()
    assert call(tokens=None) == 1 and call(lp=None) == 1 and call(n=-1) == 1
    assert call(top=33) == 1 and call(top=-1) == 1 and b"top_k" in lib.rwkv7_b200_last_error()
    assert call(ids=None) == 1 and call(top_lp=None) == 1


def test_head_logprobs_refusals(lib):
    need = C.c_size_t()
    assert lib.rwkv7_b200_head_logprobs_workspace(5, 1000, C.byref(need)) == 0 and need.value > 0
    assert lib.rwkv7_b200_head_logprobs_workspace(0, 1000, C.byref(need)) == 1
    assert lib.rwkv7_b200_head_logprobs_workspace(5, 1000, None) == 1
    lib.rwkv7_b200_head_logprobs_workspace(5, 1000, C.byref(need))

    def call(rows=5, K=64, V=1000, x=P, w=P, fmt=0, scale=None, zero=None, group=128, tokens=P, lp=P, work=P, size=need.value):
        return lib.rwkv7_b200_head_logprobs(None, rows, K, V, x, w, fmt, scale, zero, group, tokens, lp, None, None, work, size)
    assert call(rows=0) == 1 and call(K=0) == 1 and call(V=0) == 1 and call(x=None) == 1 and call(w=None) == 1
    assert call(K=48) == 2 and call(fmt=3) == 1 and call(fmt=-1) == 1
    assert call(fmt=1) == 1 and call(fmt=2) == 1 and b"scales" in lib.rwkv7_b200_last_error()
    assert call(fmt=2, scale=P, group=16) == 2
    assert call(tokens=None) == 1 and call(lp=None) == 1
    assert call(work=None) == 1 and call(size=need.value - 1) == 1 and b"workspace" in lib.rwkv7_b200_last_error()
    assert call(x=C.c_void_p((1 << 20) + 2)) == 1 and call(w=C.c_void_p((1 << 20) + 8)) == 1 and b"aligned" in lib.rwkv7_b200_last_error()


def test_linear_w4a16_group_refusals(lib):
    def call(M=1, K=64, N=4, x=P, q=P, scale=P, group=32, epi=0, y=P):
        return lib.rwkv7_b200_linear_w4a16_group(None, M, K, N, x, q, scale, None, group, epi, y, None, 0)
    assert call(M=0) == 1 and call(N=0) == 1 and call(K=0) == 1
    assert call(K=72) == 2 and call(group=16) == 2 and call(group=256) == 2 and call(group=0) == 2
    assert call(x=None) == 1 and call(q=None) == 1 and call(scale=None) == 1 and call(y=None) == 1
    assert call(epi=2) == 1 and call(epi=4) == 1 and b"epilogue" in lib.rwkv7_b200_last_error()
    assert call(q=C.c_void_p((1 << 20) + 4)) == 1
    pack, unpack = lib.rwkv7_b200_quant_pack_w4_group, lib.rwkv7_b200_quant_unpack_w4_group
    assert pack(None, 4, 40, 32, P, P, P, P) == 2 and pack(None, 4, 64, 48, P, P, P, P) == 2 and pack(None, 4, 64, 32, None, P, P, P) == 1
    assert unpack(None, 0, 64, 32, P, P, P, P) == 1 and unpack(None, 4, 64, 32, P, P, P, None) == 1


def test_exact_flag_of_the_4bit_product(lib):
    """Or-ed to a known epilogue it is none of its own; other bits, and other linear layers, stay refused.  The scratch asked for serves both forms."""
    from rwkv_lightning_cuda_b200 import lib as L
    def call(epi, K=72):
        return lib.rwkv7_b200_linear_w4a16_group(None, 1, K, 4, P, P, P, None, 32, epi, P, None, 0)
    for epi in (0, 1, 3):
        assert call(epi | L.EPI_EXACT) == 2 and b"multiple of 32" in lib.rwkv7_b200_last_error()  # (refused for its K)
    for epi in (2, 4, 32, 64):
        assert call(epi | L.EPI_EXACT, 64) == 1 and b"epilogue" in lib.rwkv7_b200_last_error()
    assert lib.rwkv7_b200_linear_w4a16(None, 1, 128, 4, P, P, P, P, L.EPI_EXACT, P) == 1
    need = C.c_size_t()
    assert lib.rwkv7_b200_linear_w4a16_group_workspace(96, 10272, 2560, C.byref(need)) == 0 and need.value > 0
    assert lib.rwkv7_b200_linear_w4a16_group_workspace(8, 10272, 2560, C.byref(need)) == 0 and need.value == 0


def test_python_layer_refuses_before_it_calls():
    """CPU tensors, wrong types, shapes and layouts: an error that names the argument (the device tensors' own checks run in the
    GPU tests)."""
    from rwkv_lightning_cuda_b200 import lib as L, ops
    z = torch.zeros(2, 8)
    for bad, text in ((lambda: ops.token_logprobs(z), "device"), (lambda: ops.token_logprobs(z[0]), "rows, V"),
                      (lambda: ops.token_logprobs(z.double()), "float32"), (lambda: ops.token_logprobs(None), "rows, V"),
                      (lambda: ops.head_logprobs(z.half(), z.half()), "device"), (lambda: ops.head_logprobs(z, z), "float16"),
                      (lambda: ops.linear_w4a16_group(z.half(), z.byte(), z.half()), "device"),
                      (lambda: ops.quant_pack_w4_group(z), "float16"), (lambda: ops.quant_unpack_w4_group(z, z), "uint8")):
        with pytest.raises(L.Rwkv7B200Error, match=text):
            bad()


def test_references_agree_with_torch():
    """The references the GPU tests compare with, against torch's own functions and against differences: the log of the
    sum has the probabilities as its derivative."""
    from tests.head_end import ref_logprobs
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(4, 50, generator=gen, dtype=torch.float64) * 3
    z[1, 7] = float("-inf")
    tok = torch.tensor([[3, -1], [7, 0], [49, 50], [0, 1]])
    lp, H, lse, ids, tlp = ref_logprobs(z, tok, 5)
    want = torch.log_softmax(z, 1)
    assert torch.allclose(lp[0, 0], want[0, 3]) and lp[0, 1] == 0 and lp[1, 0] == float("-inf") and torch.isnan(lp[2, 1])
    assert torch.allclose(lse, torch.logsumexp(z, 1)) and torch.allclose(H[0], torch.distributions.Categorical(logits=z[0]).entropy())
    top = want.topk(5, dim=1)
    assert torch.equal(ids.long(), top.indices) and torch.allclose(tlp, top.values)
    h = 1e-6
    up, down = z.clone(), z.clone()
    up[:, 11] += h
    down[:, 11] -= h
    assert torch.allclose((ref_logprobs(up)[2] - ref_logprobs(down)[2]) / (2 * h), want[:, 11].exp(), atol=1e-8)


def test_rounded_weights_of_any_zero():
    """The halves that weights with any zero count as: half((q - zero) * scale) for whole zeros, and otherwise off that product by half a step and
    2^-17 of the scale (a 32nd of the scale, rounded to half)."""
    from tests.head_end import random_w4, w4_rounded_any_zero, w4_weights
    gen = torch.Generator().manual_seed(5)
    q, s, z = random_w4(40, 256, 32, False, gen, device="cpu")
    assert torch.equal(w4_rounded_any_zero(q, s, z, 32), w4_weights(q, s, z, 32, rounded=True))
    z = (torch.rand(z.shape, generator=gen) * 16).half()
    off = (w4_rounded_any_zero(q, s, z, 32) - w4_weights(q, s, z, 32)).abs()
    allowed = w4_weights(q, s, z, 32).abs() * 2.0 ** -11 * (1 + 1e-3) + s.double()[:, torch.arange(256) // 32] * 2.0 ** -17 + 2.0 ** -25
    assert bool((off <= allowed).all()) and float(off.max()) > 0
