"""Op-level bindings: one function per ``rwkv7_b200_*`` launcher export, on torch CUDA tensors.

Names follow the reference's launcher surface (cuda/rwkv7_fast_v4_kernels.cuh).  Everything is
enqueued on the current torch stream; nothing here computes on the host.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import List, Optional, Sequence

import torch

from . import lib as L


def _s():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t: Optional[torch.Tensor]):
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensors only"
    return C.c_void_p(t.data_ptr())


def _ptr_table(ts: Sequence[torch.Tensor]):
    arr = (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])
    return arr


def wkv_fp16_seq(B, T, H, state, r, w, k, v, a, b, elapsed, w0=None):
    y = torch.empty_like(r)
    lib = L.load_library()
    Cc = H * 64
    if w0 is None:
        L.check(lib.rwkv7_b200_wkv_fp16_seq(_s(), B, T, Cc, H, _p(state), _p(r), _p(w), _p(k), _p(v), _p(a), _p(b), _p(y), _p(elapsed)))
    else:
        L.check(lib.rwkv7_b200_wkv_fp16_seq_w0(_s(), B, T, Cc, H, _p(state), _p(r), _p(w), _p(w0), _p(k), _p(v), _p(a), _p(b), _p(y), _p(elapsed)))
    return y


def wkv_fp32io16(B, T, H, state, r, w, k, v, a, b):
    y = torch.empty_like(r)
    L.check(L.load_library().rwkv7_b200_wkv_fp32io16(_s(), B, T, H * 64, H, _p(state), _p(r), _p(w), _p(k), _p(v), _p(a), _p(b), _p(y)))
    return y


def tmix_mix6(B, T, x, shift, mixes: Sequence[torch.Tensor]) -> List[torch.Tensor]:
    outs = [torch.empty_like(x) for _ in range(6)]
    L.check(L.load_library().rwkv7_b200_tmix_mix6(_s(), B, T, x.shape[-1], _p(x), _p(shift), _ptr_table(mixes), _ptr_table(outs)))
    return outs


def cmix_mix(B, T, x, shift, x_k):
    out = torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_cmix_mix(_s(), B, T, x.shape[-1], _p(x), _p(shift), _p(x_k), _p(out)))
    return out


def tmix_kk_a_gate(B, T, H, k, k_k, a0, a12, k_a):
    nk, nkk, kka = torch.empty_like(k), torch.empty_like(k), torch.empty_like(k)
    L.check(L.load_library().rwkv7_b200_tmix_kk_a_gate(_s(), B, T, H * 64, H, _p(k), _p(k_k), _p(a0), _p(a12), _p(k_a), _p(nk), _p(nkk), _p(kka)))
    return nk, nkk, kka


def tmix_lnx_rkvres_xg(B, T, H, x, r, k, v, r_k, weight, bias, g):
    out = torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_tmix_lnx_rkvres_xg(_s(), B, T, H * 64, H, _p(x), _p(r), _p(k), _p(v), _p(r_k), _p(weight), _p(bias), _p(g), _p(out)))
    return out


def tmix_vres_gate(B, T, v, v_first, v0, v12):
    out = torch.empty_like(v)
    L.check(L.load_library().rwkv7_b200_tmix_vres_gate(_s(), B, T, v.shape[-1], _p(v), _p(v_first), _p(v0), _p(v12), _p(out)))
    return out


def layer_norm_f16(x, weight, bias, eps=1e-5):
    y = torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_layer_norm_f16(_s(), x.shape[0], x.shape[1], _p(x), _p(weight), _p(bias), _p(y), eps))
    return y


def add_layer_norm_f16(x, residual, weight, bias, eps=1e-5):
    xo, y = torch.empty_like(x), torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_add_layer_norm_f16(_s(), x.shape[0], x.shape[1], _p(x), _p(residual), _p(weight), _p(bias), _p(xo), _p(y), eps))
    return xo, y


def add_last_layer_norm_f16(B, T, x, residual, weight, bias, eps=1e-5):
    y = torch.empty((B, x.shape[-1]), dtype=torch.float16, device=x.device)
    L.check(L.load_library().rwkv7_b200_add_last_layer_norm_f16(_s(), B, T, x.shape[-1], _p(x), _p(residual), _p(weight), _p(bias), _p(y), eps))
    return y


def add_layer_norm_cmix_mix_f16(B, T, x, residual, shift, weight, bias, x_k, eps=1e-5):
    xo, mixed = torch.empty_like(x), torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_add_layer_norm_cmix_mix_f16(_s(), B, T, x.shape[-1], _p(x), _p(residual), _p(shift), _p(weight), _p(bias), _p(x_k), _p(xo), _p(mixed), eps))
    return xo, mixed


def add_layer_norm_tmix_mix6_f16(B, T, x, residual, shift, weight, bias, mixes, eps=1e-5):
    xo = torch.empty_like(x)
    outs = [torch.empty_like(x) for _ in range(6)]
    L.check(L.load_library().rwkv7_b200_add_layer_norm_tmix_mix6_f16(_s(), B, T, x.shape[-1], _p(x), _p(residual), _p(shift), _p(weight), _p(bias), _ptr_table(mixes), _p(xo), _ptr_table(outs), eps))
    return xo, outs


def emb_ln0(emb, weight, bias, eps=1e-5):
    dt = L.DT_BF16 if emb.dtype == torch.bfloat16 else L.DT_F16
    out = torch.empty(emb.shape, dtype=torch.float16, device=emb.device)
    L.check(L.load_library().rwkv7_b200_emb_ln0(_s(), emb.shape[0], emb.shape[1], _p(emb), _p(weight), _p(bias), dt, _p(out), eps))
    return out


def relu_square(x):
    out = torch.empty_like(x)
    L.check(L.load_library().rwkv7_b200_relu_square(_s(), _p(x), _p(out), x.numel()))
    return out


def advance_i32(x, amount):
    L.check(L.load_library().rwkv7_b200_advance_i32(_s(), _p(x), amount, x.numel()))


def greedy_pick(logits, penalties=None, presence_penalty=0.0, repetition_penalty=0.0, penalty_decay=1.0, next_tokens=None):
    """Token ids int32 [B] = argmax(logits - penalties) per row; ``penalties`` is updated in place."""
    B, V = logits.shape
    out = torch.empty((B,), dtype=torch.int32, device=logits.device)
    L.check(L.load_library().rwkv7_b200_greedy_pick(_s(), B, V, _p(logits), _p(penalties), presence_penalty, repetition_penalty,
                                                    penalty_decay, _p(out), _p(next_tokens)))
    return out


def _out(x, N, epi):
    return torch.empty((x.shape[0], N), dtype=torch.float32 if epi == L.EPI_F32 else torch.float16, device=x.device)


def linear_f16_orig(x, weight, in_act=L.ACT_NONE, epilogue=L.EPI_NONE):
    y = _out(x, weight.shape[0], epilogue)
    L.check(L.load_library().rwkv7_b200_linear_f16_orig(_s(), x.shape[0], x.shape[1], weight.shape[0], _p(x), _p(weight), in_act, epilogue, _p(y)))
    return y


def linear_f16_orig_static(x, weight, epilogue=L.EPI_NONE, out=None):
    """linear_f16_orig for more than four rows through the entry point that allocates nothing itself
    (its split-K scratch is a fixed device array inside the library).  Pass `out` to avoid the
    allocation of the result tensor as well."""
    y = _out(x, weight.shape[0], epilogue) if out is None else out
    L.check(L.load_library().rwkv7_b200_linear_f16_orig_static(_s(), x.shape[0], x.shape[1], weight.shape[0], _p(x), _p(weight), epilogue, _p(y)))
    return y


def linear_w8a16(x, q, scale, epilogue=L.EPI_NONE):
    y = _out(x, q.shape[0], epilogue)
    L.check(L.load_library().rwkv7_b200_linear_w8a16(_s(), x.shape[0], x.shape[1], q.shape[0], _p(x), _p(q), _p(scale), epilogue, _p(y)))
    return y


def linear_w4a16(x, q, scale, zero, epilogue=L.EPI_NONE):
    y = _out(x, q.shape[0], epilogue)
    L.check(L.load_library().rwkv7_b200_linear_w4a16(_s(), x.shape[0], x.shape[1], q.shape[0], _p(x), _p(q), _p(scale), _p(zero), epilogue, _p(y)))
    return y


def quant_pack_w8(W):
    N, K = W.shape
    q = torch.empty((N, K), dtype=torch.int8, device=W.device)
    s = torch.empty((N,), dtype=torch.float16, device=W.device)
    L.check(L.load_library().rwkv7_b200_quant_pack_w8(_s(), N, K, _p(W), _p(q), _p(s)))
    return q, s


def quant_unpack_w8(q, s):
    W = torch.empty(q.shape, dtype=torch.float16, device=q.device)
    L.check(L.load_library().rwkv7_b200_quant_unpack_w8(_s(), q.shape[0], q.shape[1], _p(q), _p(s), _p(W)))
    return W


def quant_pack_w4(W):
    N, K = W.shape
    q = torch.empty((N, K // 2), dtype=torch.uint8, device=W.device)
    s = torch.empty((N, K // 128), dtype=torch.float16, device=W.device)
    z = torch.empty((N, K // 128), dtype=torch.float16, device=W.device)
    L.check(L.load_library().rwkv7_b200_quant_pack_w4(_s(), N, K, _p(W), _p(q), _p(s), _p(z)))
    return q, s, z


def quant_unpack_w4(q, s, z):
    N, K = q.shape[0], q.shape[1] * 2
    W = torch.empty((N, K), dtype=torch.float16, device=q.device)
    L.check(L.load_library().rwkv7_b200_quant_unpack_w4(_s(), N, K, _p(q), _p(s), _p(z), _p(W)))
    return W


def sample(logits, penalties=None, presence=0.0, repetition=0.0, decay=1.0, temperature=1.0, top_k=0, top_p=1.0, seed=0, offset=0,
           next_tokens=None):
    """One token per row of fp32 logits [B, V] with the sampler's rule (temperature, top-k, top-p, penalties updated in
    place); the draw is a function of (seed, offset, row).  Returns int32 [B] on the device."""
    B, V = logits.shape
    out = torch.empty((B,), dtype=torch.int32, device=logits.device)
    probs = torch.empty((B, V), dtype=torch.float32, device=logits.device)
    sp = L.Sampling(temperature, top_k, top_p, seed, offset)
    import ctypes as C
    L.check(L.load_library().rwkv7_b200_sample(_s(), B, V, _p(logits), _p(penalties), _p(probs), presence, repetition, decay,
                                                C.byref(sp), _p(out), _p(next_tokens)))
    return out


def _need(ok, message, status=1):
    if not ok:
        raise L.Rwkv7B200Error(status, message)


def _tensor(name, t, dtypes, device, shape=None, contiguous=True):
    """Checks one argument of the functions below: its type, device, shape and layout."""
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _need(False, f"{name}: {' or '.join(str(d) for d in dtypes)} tensor expected")
    if not t.is_cuda or (device is not None and t.device != device):
        _need(False, f"{name}: must be on the device of the other arguments")
    if shape is not None and t.shape != shape:
        _need(False, f"{name}: shape {tuple(t.shape)}, expected {shape}", 2)
    if contiguous and not t.is_contiguous():
        _need(False, f"{name}: must be contiguous")


# The functions below run in ten microseconds or less, so a call tests everything in one expression and looks for the argument to
# name in the error only when that fails.
_F16, _F32 = torch.float16, torch.float32


def _enqueue(dev, call, *args):
    """One library call on the current stream of ``dev``, which need not be the current device; the tensors' addresses are passed as
    integers (None: NULL), the checks have been made."""
    index = dev.index
    if index == torch.cuda.current_device():
        status = call(torch._C._cuda_getCurrentRawStream(index), *args)
    else:
        with torch.cuda.device(index):
            status = call(torch._C._cuda_getCurrentRawStream(index), *args)
    if status:
        L.check(status)


def _good(t, dtype, dev, shape):
    return t.dtype == dtype and t.device == dev and t.shape == shape and t.is_contiguous()


def _refuse_token_logprobs(logits, tokens, top_k):
    _need(isinstance(logits, torch.Tensor) and logits.dim() == 2, "token_logprobs: logits [rows, V] expected", 2)
    _tensor("token_logprobs: logits", logits, (_F32, _F16), None, contiguous=False)
    rows, V = logits.shape
    _need(rows > 0 and V > 0, "token_logprobs: logits must not be empty")
    _need((logits.stride(1) == 1 or V == 1) and (rows == 1 or logits.stride(0) >= V),
          "token_logprobs: a row's logits must be contiguous, rows must not overlap")
    if tokens is not None:
        _need(isinstance(tokens, torch.Tensor) and tokens.dim() in (1, 2), "token_logprobs: tokens [rows] or [rows, n] expected", 2)
        _tensor("token_logprobs: tokens", tokens, torch.int64, logits.device, (rows, tokens.shape[1]) if tokens.dim() == 2 else (rows,))
    _need(False, "token_logprobs: top_k outside [0, 32]")


def token_logprobs(logits, tokens=None, top_k=0):
    """Log probabilities under softmax(logits [rows, V]) (fp32 or fp16; rows may be strided): of the given ``tokens`` (int64
    [rows] or [rows, n]; an id below 0 asks for nothing and gets 0, one beyond the vocabulary NaN), and of the ``top_k``
    (at most 32) likeliest tokens, likeliest first, equal ones by index.  Returns (logprobs, entropy, lse, top_ids,
    top_logprobs): fp32 shaped like ``tokens``, fp32 [rows], fp32 [rows], int32 and fp32 [rows, top_k]; None for what was not
    asked.  -inf masks a token; a row with a NaN or +inf answers NaN."""
    ok = isinstance(logits, torch.Tensor) and logits.dim() == 2 and logits.is_cuda and (logits.dtype == _F32 or logits.dtype == _F16)
    n, logprobs, ids, top, asked = 0, None, None, None, None
    if ok:
        (rows, V), (ld, along), dev = logits.shape, logits.stride(), logits.device
        if rows == 1:
            ld = V
        ok = rows > 0 and V > 0 and (along == 1 or V == 1) and ld >= V and type(top_k) is int and 0 <= top_k <= 32
        if ok and tokens is not None:
            ok = isinstance(tokens, torch.Tensor) and tokens.dim() in (1, 2) and _good(tokens, torch.int64, dev, (rows, *tokens.shape[1:]))
    if not ok:
        _refuse_token_logprobs(logits, tokens, top_k)
    if tokens is not None:
        n, asked = tokens.numel() // rows, tokens.data_ptr()
        logprobs = torch.empty_like(tokens, dtype=_F32)
    entropy, lse = torch.empty(rows, dtype=_F32, device=dev), torch.empty(rows, dtype=_F32, device=dev)
    if top_k:
        ids, top = torch.empty(rows, top_k, dtype=torch.int32, device=dev), torch.empty(rows, top_k, dtype=_F32, device=dev)
    _enqueue(dev, L.load_library().rwkv7_b200_token_logprobs, rows, V, logits.data_ptr(), L.DT_F16 if logits.dtype == _F16 else L.DT_F32, ld,
             asked, n, top_k, logprobs.data_ptr() if asked else None, entropy.data_ptr(), lse.data_ptr(), ids.data_ptr() if top_k else None,
             top.data_ptr() if top_k else None)
    return logprobs, entropy, lse, ids, top


def _w4_group_params(what, scale, zero, rows, K, group, dev):
    _need(group in (32, 64, 128), f"{what}: groups of 32, 64 or 128", 2)
    groups = -(-K // group)
    _tensor(f"{what}: scale", scale, _F16, dev, (rows, groups))
    if zero is not None:
        _tensor(f"{what}: zero", zero, _F16, dev, (rows, groups))


def _good_w4_group(scale, zero, rows, K, group, dev):
    if group not in (32, 64, 128) or not isinstance(scale, torch.Tensor):
        return False
    shape = (rows, -(-K // group))
    return _good(scale, _F16, dev, shape) and (zero is None or (isinstance(zero, torch.Tensor) and _good(zero, _F16, dev, shape)))


_HEAD_FORMATS = {torch.float16: L.FMT_F16, torch.int8: L.FMT_W8A16, torch.uint8: L.FMT_W4A16}

@functools.lru_cache(maxsize=4096)
def _scratch_bytes(query, *sizes):
    """Bytes of scratch that the library asks for at these sizes."""
    size = C.c_size_t()
    L.check(getattr(L.load_library(), query)(*sizes, C.byref(size)))
    return size.value



def _refuse_head_logprobs(x, weight, tokens, scale, zero, group_size):
    _need(isinstance(x, torch.Tensor) and x.dim() == 2 and x.shape[0] > 0, "head_logprobs: x [rows, K] expected", 2)
    _tensor("head_logprobs: x", x, _F16, None)
    rows, K = x.shape
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2 and weight.shape[0] > 0, "head_logprobs: weight [V, K] expected", 2)
    V, fmt = weight.shape[0], _HEAD_FORMATS.get(weight.dtype, -1)
    _tensor("head_logprobs: weight", weight, tuple(_HEAD_FORMATS), x.device, (V, K // 2 if fmt == L.FMT_W4A16 else K))
    if fmt == L.FMT_W8A16:
        _tensor("head_logprobs: scale", scale, _F16, x.device, (V,))
    elif fmt == L.FMT_W4A16:
        _w4_group_params("head_logprobs", scale, zero, V, K, group_size, x.device)
    _tensor("head_logprobs: tokens", tokens, torch.int64, x.device, (rows,))
    _need(False, "head_logprobs: bad argument")


def head_logprobs(x, weight, tokens=None, scale=None, zero=None, group_size=128):
    """``token_logprobs`` of x W^T (x fp16 [rows, K]) without writing the logits: one given token per row (int64 [rows] or
    None).  ``weight`` is fp16 [V, K], int8 [V, K] with ``scale`` fp16 [V], or uint8 [V, K/2] (two 4-bit codes a byte) with
    ``scale`` and ``zero`` (None: 8) fp16 [V, ceil(K / group_size)], a weight counting as half((q - zero) * scale).  Returns (logprobs, entropy, lse), fp32 [rows]."""
    ok = isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and x.dim() == 2 and weight.dim() == 2 and x.is_cuda
    if ok:
        (rows, K), V, dev, fmt = x.shape, weight.shape[0], x.device, _HEAD_FORMATS.get(weight.dtype, -1)
        ok = (rows > 0 and V > 0 and fmt >= 0 and x.dtype == _F16 and x.is_contiguous()
              and _good(weight, weight.dtype, dev, (V, K // 2 if fmt == L.FMT_W4A16 else K))
              and (tokens is None or (isinstance(tokens, torch.Tensor) and _good(tokens, torch.int64, dev, (rows,)))))
        if ok and fmt == L.FMT_W8A16:
            ok = isinstance(scale, torch.Tensor) and _good(scale, _F16, dev, (V,))
        elif ok and fmt == L.FMT_W4A16:
            ok = _good_w4_group(scale, zero, V, K, group_size, dev)
    if not ok:
        _refuse_head_logprobs(x, weight, tokens, scale, zero, group_size)
    lib = L.load_library()
    need = _scratch_bytes("rwkv7_b200_head_logprobs_workspace", rows, V)
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    logprobs = torch.empty(rows, dtype=_F32, device=dev) if tokens is not None else None
    entropy, lse = torch.empty(rows, dtype=_F32, device=dev), torch.empty(rows, dtype=_F32, device=dev)
    _enqueue(dev, lib.rwkv7_b200_head_logprobs, rows, K, V, x.data_ptr(), weight.data_ptr(), fmt, scale.data_ptr() if fmt else None,
             zero.data_ptr() if fmt == L.FMT_W4A16 and zero is not None else None, group_size, tokens.data_ptr() if tokens is not None else None,
             logprobs.data_ptr() if tokens is not None else None, entropy.data_ptr(), lse.data_ptr(), work.data_ptr(), need)
    return logprobs, entropy, lse


def _refuse_linear_w4a16_group(x, q, scale, zero, group_size):
    _need(isinstance(x, torch.Tensor) and x.dim() == 2 and x.shape[0] > 0, "linear_w4a16_group: x [M, K] expected", 2)
    _tensor("linear_w4a16_group: x", x, _F16, None)
    _need(isinstance(q, torch.Tensor) and q.dim() == 2 and q.shape[0] > 0, "linear_w4a16_group: q [N, K/2] expected", 2)
    K, N = x.shape[1], q.shape[0]
    _tensor("linear_w4a16_group: q", q, torch.uint8, x.device, (N, K // 2))
    _w4_group_params("linear_w4a16_group", scale, zero, N, K, group_size, x.device)
    _need(False, "linear_w4a16_group: bad argument")


def linear_w4a16_group(x, q, scale, zero=None, group_size=128, epilogue=L.EPI_NONE, exact=False):
    """x W^T for 4-bit weights with group scales: W = (q - zero) * scale per group of 32, 64 or 128 inputs; x fp16 [M, K], q
    uint8 [N, K/2], scale and zero (None: 8) fp16 [N, ceil(K / group_size)]; K a multiple of 32, any M and N.  Up to 8
    rows no weight is rounded; with more a weight counts as half((q - zero) * scale), unless ``exact`` asks for weights that are not
    rounded there either (at twice the products).  Zeros need not be whole numbers; with more than 8
    rows other ones (from -32 on) put a weight off by 2^-17 of its scale (``exact``: 2^-15) at most."""
    ok = isinstance(x, torch.Tensor) and isinstance(q, torch.Tensor) and x.dim() == 2 and q.dim() == 2 and x.is_cuda
    if ok:
        (M, K), N, dev = x.shape, q.shape[0], x.device
        ok = (M > 0 and N > 0 and x.dtype == _F16 and x.is_contiguous() and _good(q, torch.uint8, dev, (N, K // 2))
              and _good_w4_group(scale, zero, N, K, group_size, dev))
    if not ok:
        _refuse_linear_w4a16_group(x, q, scale, zero, group_size)
    y = torch.empty(M, N, dtype=_F32 if epilogue == L.EPI_F32 else _F16, device=dev)
    need, work = 0, None
    if M > 8:
        need = _scratch_bytes("rwkv7_b200_linear_w4a16_group_workspace", M, K, N)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _enqueue(dev, L.load_library().rwkv7_b200_linear_w4a16_group, M, K, N, x.data_ptr(), q.data_ptr(), scale.data_ptr(),
             None if zero is None else zero.data_ptr(), group_size, epilogue | L.EPI_EXACT if exact else epilogue, y.data_ptr(), work.data_ptr() if need else None, need)
    return y


def quant_pack_w4_group(W, group_size=128, symmetric=False):
    """4-bit codes, scales and zeros (None when ``symmetric``) of W fp16 [N, K] over groups of ``group_size`` inputs."""
    _need(isinstance(W, torch.Tensor) and W.dim() == 2, "quant_pack_w4_group: W [N, K] expected", 2)
    _tensor("quant_pack_w4_group: W", W, torch.float16, None)
    N, K = W.shape
    _need(group_size in (32, 64, 128), "quant_pack_w4_group: groups of 32, 64 or 128", 2)
    with torch.cuda.device(W.device):
        q = torch.empty((N, K // 2), dtype=torch.uint8, device=W.device)
        s = torch.empty((N, -(-K // group_size)), dtype=torch.float16, device=W.device)
        z = None if symmetric else torch.empty_like(s)
        L.check(L.load_library().rwkv7_b200_quant_pack_w4_group(_s(), N, K, group_size, _p(W), _p(q), _p(s), _p(z)))
    return q, s, z


def quant_unpack_w4_group(q, scale, zero=None, group_size=128):
    """The weights that the codes stand for, rounded to fp16 [N, K]."""
    _need(isinstance(q, torch.Tensor) and q.dim() == 2, "quant_unpack_w4_group: q [N, K/2] expected", 2)
    _tensor("quant_unpack_w4_group: q", q, torch.uint8, None)
    N, K = q.shape[0], q.shape[1] * 2
    _w4_group_params("quant_unpack_w4_group", scale, zero, N, K, group_size, q.device)
    with torch.cuda.device(q.device):
        W = torch.empty((N, K), dtype=torch.float16, device=q.device)
        L.check(L.load_library().rwkv7_b200_quant_unpack_w4_group(_s(), N, K, group_size, _p(q), _p(scale), _p(zero), _p(W)))
    return W
