"""forward_score: a prompt's log probabilities from the model, against the model's own logits and against its forward step by step."""
import pytest
import torch

from oracle import oracle as orc
from oracle.parity import TINY, build_pair
from tests.head_end import U16, ref_logprobs, softmax_tolerance

pytestmark = pytest.mark.gpu

LOGITS = 2e-2  # how far two routes through the layers may move a logit (the model tests' tolerance)


def prompt(B, T, vocab, seed=0):
    return torch.randint(0, vocab, (B, T), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("fmt", [orc.FMT_F16, orc.FMT_W8A16, orc.FMT_W4A16])
@pytest.mark.parametrize("B,T,wkv32", [(1, 1, False), (1, 2, False), (2, 3, True), (1, 9, False), (3, 40, True), (1, 130, False)])
def test_last_position_agrees_with_the_logits_of_the_same_call(fmt, B, T, wkv32):
    """The last position's answers follow from the logits that the same call returns, but for those being rounded to half; the state is the
    one forward_prefill leaves."""
    from rwkv_lightning_cuda_b200 import backend as bk
    d, _, gm = build_pair(fmt, wkv32, oracle_model=False)
    tok = prompt(B, T, d.vocab)
    want = torch.roll(tok, -1, 1)
    want[:, -1] = 5
    st, lg = gm.create_state(B), bk.DeviceLogits()
    lp, H = gm.forward_score(tok, st, want, lg)
    ref = ref_logprobs(lg.values, want[:, -1])
    biggest = float(lg.values.abs().max())
    tol = softmax_tolerance(d.vocab, biggest, biggest * U16)
    assert float((lp[:, -1].cpu().double() - ref[0]).abs().max()) <= tol
    # d entropy / d logit is at most p (|log p| + entropy) <= 1 / e + entropy, summed over moves of half a step each
    assert float((H[:, -1].cpu().double() - ref[1]).abs().max()) <= (2 * float(ref[1].max()) + 1) * tol
    plain, pl = gm.create_state(B), bk.DeviceLogits()
    gm.forward_prefill(tok, plain, pl)
    if B * T > 4:  # (up to four one-token rows forward takes the fused decode kernels)
        assert torch.equal(st.shift, plain.shift) and torch.equal(st.wkv_state, plain.wkv_state) and torch.equal(lg.values, pl.values)
    else:
        assert float((lg.values - pl.values).abs().max()) <= LOGITS
    assert st.elapsed.tolist() == [T] * B
    gm.close()


def test_every_position_against_single_steps():
    """Scored at once and fed token by token: the same distribution at every position; targets below 0 answer 0."""
    from rwkv_lightning_cuda_b200 import backend as bk
    d, _, gm = build_pair(orc.FMT_F16, False, oracle_model=False)
    B, T = 2, 12
    tok = prompt(B, T, d.vocab, 3)
    st = gm.create_state(B)
    lp, H = gm.forward_score(tok, st)
    assert lp[:, -1].tolist() == [0.0, 0.0]
    one, lg = gm.create_state(B), bk.DeviceLogits()
    for t in range(T):
        gm.forward_decode(tok[:, t].tolist(), one, lg)
        ref = ref_logprobs(lg.values, tok[:, t + 1] if t + 1 < T else None)
        if t + 1 < T:
            assert float((lp[:, t].cpu().double() - ref[0]).abs().max()) <= 2 * LOGITS
        assert float((H[:, t].cpu().double() - ref[1]).abs().max()) <= (2 * float(ref[1].max()) + 1) * LOGITS
    gm.close()


def test_chunks_and_streams_and_repeats():
    """A prompt scored in two chunks on a side stream equals itself scored again, position for position, and goes on where the first left off."""
    d, _, gm = build_pair(orc.FMT_F16, True, oracle_model=False)
    tok = prompt(1, 100, d.vocab, 4)
    outs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            st = gm.create_state(1)
            want = torch.roll(tok, -1, 1)
            a = gm.forward_score(tok[:, :36], st, want[:, :36])[0]
            b = gm.forward_score(tok[:, 36:], st, want[:, 36:])[0]
            outs.append(torch.cat([a, b], 1))
        stream.synchronize()
    assert torch.equal(outs[0], outs[1])
    st = gm.create_state(1)
    whole = gm.forward_score(tok, st, torch.roll(tok, -1, 1))[0]
    assert float((whole - outs[0]).abs().max()) <= 2 * LOGITS
    gm.close()


def test_refusals_leave_the_state_alone():
    from rwkv_lightning_cuda_b200 import lib as L
    d, _, gm = build_pair(orc.FMT_F16, False, oracle_model=False)
    st = gm.create_state(2)
    tok = prompt(2, 5, d.vocab)
    for bad, text in ((lambda: gm.forward_score(tok, st, tok[:, :4]), "shape"), (lambda: gm.forward_score(tok[:1], st), "batch size"),
                      (lambda: gm.forward_score(tok, st, tok + d.vocab), "out of range"), (lambda: gm.forward_score(tok - d.vocab, st), "out of range"),
                      (lambda: gm.forward_score([[1, 2], [3]], st), "same length")):
        with pytest.raises(L.Rwkv7B200Error, match=text):
            bad()
    assert st.elapsed.tolist() == [0, 0]
    gm.close()


def test_wide_vocabulary_model():
    """The 65536-token head at a small width: the tensor-core route (100 rows) and the few-rows one."""
    from rwkv_lightning_cuda_b200 import backend as bk
    d, _, gm = build_pair(orc.FMT_W4A16, False, oracle_model=False, dims=dict(TINY, layers=1, vocab=65536))
    for B, T in ((1, 100), (2, 2)):
        tok = prompt(B, T, d.vocab, T)
        st, lg = gm.create_state(B), bk.DeviceLogits()
        want = torch.roll(tok, -1, 1)
        lp, H = gm.forward_score(tok, st, want, lg)
        ref = ref_logprobs(lg.values, want[:, -1])
        biggest = float(lg.values.abs().max())
        assert float((lp[:, -1].cpu().double() - ref[0]).abs().max()) <= softmax_tolerance(d.vocab, biggest, biggest * U16)
        assert bool(torch.isfinite(lp).all()) and bool((H > 0).all())
    gm.close()


def test_decode_step_on_a_large_fp16_head():
    """One token on an fp16 head of 134 MB, whose logits are streamed into scratch: the answers follow from the logits of the same call, and a
    prompt scored one token a call agrees with the prompt scored at once."""
    from rwkv_lightning_cuda_b200 import backend as bk
    d, _, gm = build_pair(orc.FMT_F16, False, oracle_model=False, dims=dict(TINY, layers=1, channels=1024, ffn=1024, vocab=65536))
    T = 5
    tok = prompt(1, T, d.vocab, 2)
    want = torch.roll(tok, -1, 1)
    whole, H = gm.forward_score(tok, gm.create_state(1), want)
    st, lg = gm.create_state(1), bk.DeviceLogits()
    for t in range(T):
        lp, h = gm.forward_score(tok[:, t:t + 1], st, want[:, t:t + 1], lg)
        ref = ref_logprobs(lg.values, want[:, t])
        biggest = float(lg.values.abs().max())
        tol = softmax_tolerance(d.vocab, biggest, biggest * U16)
        assert float((lp[:, 0].cpu().double() - ref[0]).abs().max()) <= tol
        assert float((h[:, 0].cpu().double() - ref[1]).abs().max()) <= (2 * float(ref[1].max()) + 1) * tol
        assert float((lp[:, 0] - whole[:, t]).abs().max()) <= 2 * LOGITS
        assert float((h[:, 0] - H[:, t]).abs().max()) <= (2 * float(ref[1].max()) + 1) * LOGITS
    assert st.elapsed.tolist() == [T]
    gm.close()
