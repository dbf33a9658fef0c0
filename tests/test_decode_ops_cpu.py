"""Refusals of the decode step's operators, without a GPU: every argument check runs before the
first CUDA call."""

import ctypes

import pytest
import torch

from newt_b200 import ops
from newt_b200.runtime import abi

P = 1 << 12     # a pointer that is never followed: every call below is refused or empty


def _cache(**changes):
    fields = dict(k=P, v=P, ks=P, vs=P, pages=8, heads=2, page=16, d=64, kp=2048, kh=1024, kt=64,
                  vp=2048, vh=1024, vt=64, kss=2, vss=2)
    fields.update(changes)
    return abi.KV_CACHE.pack(*fields.values())


def _append(cache=None, k=P, v=P, tokens=4, table=P, max_pages=4, starts=P, offsets=P, batch=2,
            max_new=2, dtype=abi.BF16):
    return abi.load().nb200_kv_append(cache or _cache(), k, v, tokens, 128, 64, 128, 64, table, 4,
                                      max_pages, starts, offsets, batch, max_new, dtype, None)


def _attend(cache=None, q=P, out=2 * P, batch=2, queries=1, heads=4, table=P, max_pages=4, lengths=P,
            scale=0.125, window=0, sinks=0, dtype=abi.BF16, workspace=P, size=1 << 40):
    return abi.load().nb200_kv_attention(q, cache or _cache(), out, batch, queries, heads, 256, 256,
                                         64, 256, 256, 64, table, 4, max_pages, lengths, scale,
                                         window, sinks, dtype, workspace, size, None)


def _rms(x=P, res=None, w=P, out=P, res_out=None, scales=None, rows=2, n=64, group=0, eps=1e-6,
         dtype=abi.BF16, out_dtype=abi.BF16):
    return abi.load().nb200_rmsnorm(x, res, w, out, res_out, scales, rows, n, n, n, n, n, 1, group,
                                    eps, dtype, out_dtype, None)


def _score(logits=P, tokens=P, logprob=P, best=None, index=None, rows=2, vocab=100, top=0, inv=1.0,
           dtype=abi.F32):
    return abi.load().nb200_token_logprobs(logits, tokens, logprob, P, P, best, index, rows, vocab,
                                           vocab, top, inv, dtype, None)


def _grad(logits=P, tokens=P, lse=P, entropy=P, g=P, ge=P, out=P, rows=2, vocab=100, inv=1.0,
          dtype=abi.F32):
    return abi.load().nb200_token_logprobs_bwd(logits, tokens, lse, entropy, g, ge, out, rows,
                                               vocab, vocab, vocab, inv, dtype, None)


@pytest.mark.parametrize("call, code, word", [
    (lambda: _rms(rows=-1), abi.E_INVALID, "negative"),
    (lambda: _rms(rows=1 << 31), abi.E_INVALID, "int32"),
    (lambda: _rms(n=32769), abi.E_UNSUPPORTED, "32768"),
    (lambda: _rms(dtype=7, out_dtype=7), abi.E_INVALID, "dtype"),
    (lambda: _rms(dtype=abi.E4M3, out_dtype=abi.E4M3), abi.E_INVALID, "dtype"),
    (lambda: _rms(out_dtype=abi.F16), abi.E_INVALID, "e4m3"),
    (lambda: _rms(out_dtype=abi.E4M3), abi.E_INVALID, "null"),
    (lambda: _rms(out_dtype=abi.E4M3, scales=P, group=48), abi.E_INVALID, "group"),
    (lambda: _rms(group=64), abi.E_INVALID, "e4m3"),
    (lambda: _rms(eps=-1.0), abi.E_INVALID, "eps"),
    (lambda: _rms(eps=float("nan")), abi.E_INVALID, "eps"),
    (lambda: _rms(w=None), abi.E_INVALID, "null"),
    (lambda: _append(_cache(d=96)), abi.E_UNSUPPORTED, "head_dim"),
    (lambda: _append(_cache(page=24)), abi.E_UNSUPPORTED, "pages of"),
    (lambda: _append(_cache(heads=0)), abi.E_INVALID, "heads"),
    (lambda: _append(_cache(k=0)), abi.E_INVALID, "null"),
    (lambda: _append(_cache(k=P + 8)), abi.E_UNSUPPORTED, "aligned"),
    (lambda: _append(_cache(vh=1032)), abi.E_UNSUPPORTED, "strides"),
    (lambda: _append(_cache(kt=48)), abi.E_INVALID, "shorter"),
    (lambda: _append(_cache(kss=1)), abi.E_INVALID, "scales"),
    (lambda: _append(dtype=abi.F32), abi.E_UNSUPPORTED, "dtype"),
    (lambda: _append(tokens=-1), abi.E_INVALID, "extent"),
    (lambda: _append(offsets=None), abi.E_INVALID, "null"),
    (lambda: _append(batch=1 << 30, max_new=1 << 20), abi.E_UNSUPPORTED, "sequences"),
    (lambda: _attend(_cache(d=32)), abi.E_UNSUPPORTED, "head_dim"),
    (lambda: _attend(dtype=abi.F32), abi.E_UNSUPPORTED, "dtype"),
    (lambda: _attend(heads=3), abi.E_INVALID, "heads"),
    (lambda: _attend(window=-1), abi.E_INVALID, "window"),
    (lambda: _attend(sinks=-1), abi.E_INVALID, "sinks"),
    (lambda: _attend(scale=0.0), abi.E_INVALID, "scale"),
    (lambda: _attend(scale=float("inf")), abi.E_INVALID, "scale"),
    (lambda: _attend(q=None), abi.E_INVALID, "null"),
    (lambda: _attend(lengths=None), abi.E_INVALID, "null"),
    (lambda: _attend(out=P), abi.E_INVALID, "must not be q"),
    (lambda: _attend(max_pages=1 << 40), abi.E_INVALID, "extent"),
    (lambda: _attend(max_pages=400, workspace=None), abi.E_INVALID, "workspace"),
    (lambda: _attend(max_pages=400, size=1000), abi.E_INVALID, "workspace"),
    (lambda: _attend(max_pages=400, workspace=P + 8), abi.E_INVALID, "workspace"),
    (lambda: _attend(_cache(pages=0)), abi.E_INVALID, "no pages"),
    (lambda: _score(vocab=0), abi.E_INVALID, "vocabulary"),
    (lambda: _score(top=33, best=P, index=P), abi.E_UNSUPPORTED, "alternatives"),
    (lambda: _score(top=20, vocab=19, best=P, index=P), abi.E_INVALID, "alternatives"),
    (lambda: _score(top=2), abi.E_INVALID, "null"),
    (lambda: _score(tokens=None), abi.E_INVALID, "null"),
    (lambda: _score(inv=0.0), abi.E_INVALID, "temperature"),
    (lambda: _score(inv=float("nan")), abi.E_INVALID, "temperature"),
    (lambda: _score(dtype=abi.E4M3), abi.E_INVALID, "dtype"),
    (lambda: _score(rows=-1), abi.E_INVALID, "negative"),
    (lambda: _grad(lse=None), abi.E_INVALID, "null"),
    (lambda: _grad(entropy=None), abi.E_INVALID, "null"),
    (lambda: _grad(tokens=None), abi.E_INVALID, "null"),
    (lambda: _grad(inv=float("inf")), abi.E_INVALID, "temperature"),
])
def test_the_library_refuses(call, code, word):
    assert call() == code
    assert word in abi.last_error()


def test_empty_calls_do_nothing():
    assert _rms(x=None, w=None, out=None, rows=0) == 0
    assert _append(batch=0) == 0 and _append(tokens=0) == 0 and _append(max_new=0) == 0
    assert _append(max_pages=0) == 0
    assert _attend(batch=0) == 0 and _attend(queries=0) == 0
    assert _score(rows=0) == 0 and _grad(rows=0) == 0 and _grad(vocab=0) == 0


def test_the_packed_cache_is_the_header_struct():
    assert abi.KV_CACHE.size == 4 * ctypes.sizeof(ctypes.c_void_p) + 12 * 8


def _tensors():
    x, w = torch.zeros(4, 64), torch.zeros(64)
    cache = ops.new_kv_cache(8, 2, 16, 64, device="cpu")
    kv = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 4, dtype=torch.int32)
    lengths = torch.zeros(2, dtype=torch.int32)
    offsets = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    return x, w, cache, kv, table, lengths, offsets, q


def test_python_refuses_tensors_that_are_not_on_the_gpu():
    x, w, cache, kv, table, lengths, offsets, q = _tensors()
    for call in (lambda: ops.rmsnorm(x, w),
                 lambda: ops.kv_append(cache, kv, kv, table, lengths, offsets, 1),
                 lambda: ops.kv_attention(q, cache, table, lengths),
                 lambda: ops.token_logprobs(x, torch.zeros(4, dtype=torch.int64)),
                 lambda: ops.token_logprobs_backward(x, None, w[:4], w[:4])):
        with pytest.raises(TypeError, match="must be a CUDA tensor"):
            call()


@pytest.mark.parametrize("error, match, call", [
    (ValueError, "shape", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w[:32])),
    (TypeError, "expected", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w.half())),
    (ValueError, "rows", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(w, w)),
    (TypeError, "rmsnorm", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x.double(), w.double())),
    (TypeError, "output", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, out_dtype=torch.half)),
    (ValueError, "group", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, out_dtype=ops.E4M3,
                                                                     group=48)),
    (ValueError, "e4m3", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, group=64)),
    (ValueError, "stride", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(torch.zeros(64, 4).t(), w)),
    (ValueError, "residual", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, residual_out=x)),
    (ValueError, "shape", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, residual=x[:2])),
    (ValueError, "share", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(x, w, out=w.expand(4, 64))),
    (ValueError, "share", lambda x, w, c, kv, t, n, o, q: ops.rmsnorm(
        x, w, residual=x, residual_out=w.expand(4, 64))),
    (ValueError, "share", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(
        q, c, t, n, out=q[:1].expand(2, 1, 4, 64))),
    (ValueError, "share", lambda x, w, c, kv, t, n, o, q: ops.token_logprobs_backward(
        x, None, w[:4], w[:4], out=w.expand(4, 64))),
    (ValueError, "'k'", lambda x, w, c, kv, t, n, o, q: ops.kv_append(c, kv[:, :1], kv, t, n, o, 1)),
    (TypeError, "kv_append", lambda x, w, c, kv, t, n, o, q: ops.kv_append(c, kv.float(), kv.float(),
                                                                          t, n, o, 1)),
    (TypeError, "'v'", lambda x, w, c, kv, t, n, o, q: ops.kv_append(c, kv, kv.half(), t, n, o, 1)),
    (ValueError, "offsets", lambda x, w, c, kv, t, n, o, q: ops.kv_append(c, kv, kv, t, n, n, 1)),
    (TypeError, "page_table", lambda x, w, c, kv, t, n, o, q: ops.kv_append(c, kv, kv, t.long(), n,
                                                                           o, 1)),
    (ValueError, "page_table", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(q, c, t[:1], n)),
    (TypeError, "lengths", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(q, c, t, n.long())),
    (ValueError, "head_dim", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(q[..., :32], c, t, n)),
    (TypeError, "kv_attention", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(q.float(), c, t, n)),
    (TypeError, "cache", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(
        q, c._replace(k=c.k.view(torch.uint8)), t, n)),
    (ValueError, "k_scales", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(
        q, c._replace(k_scales=c.k_scales[:4]), t, n)),
    (ValueError, "unit stride", lambda x, w, c, kv, t, n, o, q: ops.kv_attention(
        q, c._replace(k=torch.zeros(8, 2, 64, 16, dtype=torch.uint8).view(ops.E4M3).transpose(2, 3)),
        t, n)),
    (ValueError, "alternatives", lambda x, w, c, kv, t, n, o, q: ops.token_logprobs(x, top=33)),
    (TypeError, "tokens", lambda x, w, c, kv, t, n, o, q: ops.token_logprobs(
        x, torch.zeros(4, dtype=torch.int32))),
    (TypeError, "logits", lambda x, w, c, kv, t, n, o, q: ops.token_logprobs(x.double())),
    (ValueError, "lse", lambda x, w, c, kv, t, n, o, q: ops.token_logprobs_backward(x, None, w, w)),
])
def test_python_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call(*_tensors())
