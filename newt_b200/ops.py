"""Operators of a served language model's step, on torch CUDA tensors: the norm between its
layers, the 8-bit key / value cache with the attention that reads it, and the log probabilities
of the tokens it answers with.

    from newt_b200 import ops

    y, _, h = ops.rmsnorm(x, weight, residual=h)
    cache = ops.new_kv_cache(pages=4096, heads=8, page_size=64, head_dim=128)
    ops.kv_append(cache, k, v, page_table, starts, offsets, max_new=1)
    o = ops.kv_attention(q, cache, page_table, lengths)
    scores = ops.token_logprobs(logits, tokens, top=20)

Each is one entry point of libnewt_b200.so (include/newt_b200.h holds the exact definitions) on
torch's current stream.  Like the operator API's launcher they refuse tensors that are not on the
current CUDA device.  Outputs that are not given, and the workspace of `kv_attention`, are fresh
tensors of torch's caching allocator on the current stream, so calls on different streams share
nothing.

`token_logprobs` of logits that require a gradient is recorded for autograd; its gradient is also
there as a function of its own.  The others have no backward pass: where gradients are enabled they
refuse tensors that require one.  Tensors that a call writes over count as modified in place.
"""

from typing import NamedTuple, Optional

import torch
from torch.autograd.graph import increment_version

from .runtime import abi

E4M3 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_HALVES = (torch.bfloat16, torch.float16)
_CODES = {torch.float32: abi.F32, torch.float16: abi.F16, torch.bfloat16: abi.BF16, E4M3: abi.E4M3}


class RmsNorm(NamedTuple):
    out: torch.Tensor
    scales: Optional[torch.Tensor]      # of an e4m3 output
    residual: Optional[torch.Tensor]    # x + residual, where a residual was given


class TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


class KVCache(NamedTuple):
    """Paged keys and values in e4m3: k, v are [pages, heads, page_size, head_dim] (any strides
    that are multiples of 16, unit stride along head_dim), the scales fp32 [pages, heads]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def new_kv_cache(pages, heads, page_size, head_dim, device=None):
    """An empty cache on the current CUDA device: all zeros, every scale 1."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    shape = (pages, heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3) for _ in range(2))
    return KVCache(k, v, torch.ones(pages, heads, device=device),
                   torch.ones(pages, heads, device=device))


# The checks below run on every call of a step whose kernels take a few microseconds: they compare
# first and word the complaint only when there is one.

_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _launch_stream(names, *tensors):
    """The current stream's handle, once every tensor given (None: not given) is seen to be a CUDA
    tensor of the current device."""
    first = tensors[0].get_device()
    if first >= 0 and first == _device():
        for t in tensors:
            if t is not None and t.get_device() != first:
                break
        else:
            return _stream(first)
    for name, t in zip(names.split(), tensors):
        if t is None:
            continue
        if not t.is_cuda:
            raise TypeError(f"argument '{name}' must be a CUDA tensor")
        if t.get_device() != _device():
            raise ValueError(f"tensor '{name}' is on {t.device} but the current device is "
                             f"cuda:{_device()}; newt launches on the current device")
    raise AssertionError("a tensor changed its device")


def _refuse(name, t, shape, dtype):
    """Says what is wrong with a tensor that is not of this shape and type, rows dense."""
    if t.shape != shape:
        raise ValueError(f"'{name}' has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"'{name}' is {t.dtype}, expected {dtype}")
    raise ValueError(f"'{name}' must have unit stride along its last dimension")


def _rows(name, t, shape, dtype):
    """Rows may lie anywhere, the elements of a row side by side."""
    if t.shape != shape or t.dtype is not dtype or (t.stride(-1) != 1 and shape[-1] > 1):
        _refuse(name, t, shape, dtype)


def _written(name, t, shape, dtype):
    """The same for a tensor that a kernel writes: no two elements in one place."""
    _rows(name, t, shape, dtype)
    if 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(shape, t.stride())):
        raise ValueError(f"'{name}' has elements that share their memory (strides {t.stride()})")


def _vector(name, t, length, dtype):
    if t.shape != (length,) or t.dtype is not dtype or not t.is_contiguous():
        _refuse(name, t, (length,), dtype)


def _no_backward(names, *tensors):
    """Refuses what would lose a gradient without a word."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            name = next(name for name, other in zip(names.split(), tensors) if other is t)
            raise RuntimeError(f"tensor '{name}' requires a gradient, but this operator has no backward "
                               "pass; call it under torch.no_grad() or give it a detached tensor")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fresh(x, dtype):
    """A contiguous tensor of x's shape (empty_like is the quicker call, but keeps x's strides)."""
    return torch.empty_like(x, dtype=dtype) if x.is_contiguous() else x.new_empty(x.shape, dtype=dtype)


def rmsnorm(x, weight, residual=None, eps=1e-6, out_dtype=None, group=0, out=None, scales=None,
            residual_out=None):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight, over the rows of [rows, n] tensors
    (fp32, fp16 or bf16; n up to 32768).  Returns (out, scales, residual).

    `out_dtype` None: out = y in x's type.  torch.float8_e4m3fn: out = y / scale in 8 bits with
    scale = max|y| / 448 over the row (`group` 0; scales [rows, 1]) or over every `group` of 32, 64
    or 128 columns (scales [rows, ceil(n / group)]).  With a residual, h comes back in x's type.
    `out` and `residual_out` may be x and residual themselves.  It has no backward pass."""
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2:
        raise ValueError(f"'x' must be [rows, n], got {tuple(shape)}")
    rows, n = shape
    if dtype not in _FLOATS:
        raise TypeError(f"rmsnorm: {dtype} (fp32, fp16 or bf16)")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype is not E4M3 and out_dtype is not dtype:
        raise TypeError(f"rmsnorm: the output is {dtype} or float8_e4m3fn, not {out_dtype}")
    _rows("x", x, shape, dtype)
    _vector("weight", weight, n, dtype)
    _no_backward("x weight residual out scales residual_out", x, weight, residual, out, scales, residual_out)
    given = None
    if out is not None or scales is not None or residual_out is not None:
        given = [t for t in (out, scales, residual_out) if t is not None]
    if out is None:
        out = _fresh(x, out_dtype)
    else:
        _written("out", out, shape, out_dtype)
    scale_stride = residual_stride = residual_out_stride = 0
    if out_dtype is E4M3:
        if group not in (0, 32, 64, 128):
            raise ValueError(f"rmsnorm: group {group} (0: one scale per row; 32, 64, 128 columns)")
        columns = -(-n // group) if group else 1
        if scales is None:
            scales = x.new_empty((rows, columns), dtype=torch.float32)
            scale_stride = columns
        else:
            _written("scales", scales, (rows, columns), torch.float32)
            scale_stride = scales.stride(0)
    elif group or scales is not None:
        raise ValueError("rmsnorm: scales and groups go with an e4m3 output")
    if residual is not None:
        _rows("residual", residual, shape, dtype)
        residual_stride = residual.stride(0)
        if residual_out is None:
            residual_out = _fresh(x, dtype)
        else:
            _written("residual_out", residual_out, shape, dtype)
        residual_out_stride = residual_out.stride(0)
    elif residual_out is not None:
        raise ValueError("rmsnorm: 'residual_out' goes with a residual")
    stream = _launch_stream("x weight residual out scales residual_out", x, weight, residual, out,
                            scales, residual_out)
    abi.check(abi.load().nb200_rmsnorm(
        x.data_ptr(), _ptr(residual), weight.data_ptr(), out.data_ptr(), _ptr(residual_out),
        _ptr(scales), rows, n, x.stride(0), residual_stride, out.stride(0), residual_out_stride,
        scale_stride, group, eps, _CODES[dtype], _CODES[out_dtype], stream))
    if given:
        increment_version(given)
    return RmsNorm(out, scales, residual_out)


def _pack_cache(cache):
    """nb200_kv_cache of a KVCache, after its shapes and types have been looked at."""
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 4:
        raise ValueError(f"'cache.k' must be [pages, heads, page_size, head_dim], got {tuple(shape)}")
    pages, heads, page, d = shape
    if v.shape != shape:
        raise ValueError(f"'cache.v' has shape {tuple(v.shape)}, 'cache.k' {tuple(shape)}")
    if k.dtype is not E4M3 or v.dtype is not E4M3:
        raise TypeError(f"the cache holds {k.dtype} and {v.dtype}, expected float8_e4m3fn")
    of_scales = (pages, heads)
    _rows("cache.k_scales", ks, of_scales, torch.float32)
    _rows("cache.v_scales", vs, of_scales, torch.float32)
    kp, kh, kt, ku = k.stride()
    vp, vh, vt, vu = v.stride()
    if ku != 1 or vu != 1:
        raise ValueError("the cache must have unit stride along head_dim")
    ksp, vsp = ks.stride(0), vs.stride(0)
    if pages <= 1 or heads <= 1:
        # the stride of a dimension of one element is never used: torch may say anything there
        dense = page * d
        if heads <= 1:
            kh = vh = dense
        if pages <= 1:
            kp = vp = heads * dense
            ksp = vsp = heads
    return abi.KV_CACHE.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads,
                             page, d, kp, kh, kt, vp, vh, vt, ksp, vsp)


def _page_table(table, batch):
    shape = table.shape
    if len(shape) != 2 or shape[0] != batch:
        raise ValueError(f"'page_table' has shape {tuple(shape)}, expected ({batch}, pages)")
    _rows("page_table", table, shape, torch.int32)


def kv_append(cache, k, v, page_table, starts, offsets, max_new):
    """Writes new keys and values into the cache, in place.

    k, v: [tokens, heads, head_dim] (fp16 or bf16), the new tokens of all sequences, one sequence
    after another; sequence b brings rows offsets[b] .. offsets[b + 1) (int32, [batch + 1]) and had
    starts[b] tokens before (int32).  page_table: int32 [batch, pages], the pages of each sequence
    in order.  max_new: at least the most new tokens of one sequence.

    Scales are powers of two, one per page and head; a page that holds older tokens keeps its scale
    or gets a larger one, to which the older tokens are then brought.  Sequences must not share the
    pages they write to.  Tokens whose page the table lacks are not written.  It has no backward
    pass."""
    packed = _pack_cache(cache)
    heads, d = cache.k.shape[1], cache.k.shape[3]
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or shape[1] != heads or shape[2] != d:
        raise ValueError(f"'k' has shape {tuple(shape)}, expected (tokens, {heads}, {d})")
    if dtype not in _HALVES:
        raise TypeError(f"kv_append: {dtype} (fp16 or bf16)")
    _rows("k", k, shape, dtype)
    _rows("v", v, shape, dtype)
    batch = starts.shape[0]
    _vector("starts", starts, batch, torch.int32)
    _vector("offsets", offsets, batch + 1, torch.int32)
    _page_table(page_table, batch)
    _no_backward("k v cache.k_scales cache.v_scales", k, v, cache.k_scales, cache.v_scales)
    stream = _launch_stream(
        "k v page_table starts offsets cache.k cache.v cache.k_scales cache.v_scales", k, v,
        page_table, starts, offsets, cache.k, cache.v, cache.k_scales, cache.v_scales)
    abi.check(abi.load().nb200_kv_append(
        packed, k.data_ptr(), v.data_ptr(), shape[0], k.stride(0), k.stride(1), v.stride(0),
        v.stride(1), page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
        starts.data_ptr(), offsets.data_ptr(), batch, max_new, _CODES[dtype], stream))
    increment_version(cache)


def kv_attention(q, cache, page_table, lengths, scale=None, window=0, sinks=0, out=None):
    """Attention of the newest tokens of each sequence over the cache.

    q: [batch, queries, heads, head_dim] (fp16 or bf16); heads is a multiple of the cache's heads.
    lengths: int32 [batch], the tokens of each sequence in the cache, the new ones among them: query
    i of sequence b stands at position lengths[b] - queries + i and sees the tokens up to its own,
    with `window` > 0 only the last `window` of them and the first `sinks` of the sequence.  A query
    that sees nothing gives zeros.  scale: 1 / sqrt(head_dim) if not given.  `out` must not be q.  It has
    no backward pass."""
    packed = _pack_cache(cache)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 4:
        raise ValueError(f"'q' must be [batch, queries, heads, head_dim], got {tuple(shape)}")
    batch, queries, heads, d = shape
    if d != cache.k.shape[3]:
        raise ValueError(f"'q' has head_dim {d}, the cache {cache.k.shape[3]}")
    if dtype not in _HALVES:
        raise TypeError(f"kv_attention: {dtype} (fp16 or bf16)")
    _rows("q", q, shape, dtype)
    _vector("lengths", lengths, batch, torch.int32)
    _page_table(page_table, batch)
    _no_backward("q cache.k_scales cache.v_scales out", q, cache.k_scales, cache.v_scales, out)
    given = out is not None
    if given:
        _written("out", out, shape, dtype)
    else:
        out = _fresh(q, dtype)
    stream = _launch_stream(
        "q page_table lengths out cache.k cache.v cache.k_scales cache.v_scales", q, page_table,
        lengths, out, cache.k, cache.v, cache.k_scales, cache.v_scales)
    lib = abi.load()
    code, pages = _CODES[dtype], page_table.shape[1]
    need = lib.nb200_kv_attention_workspace_bytes(packed, batch, queries, heads, pages, code)
    ws = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    qb, qt, qh, _ = q.stride()
    ob, ot, oh, _ = out.stride()
    abi.check(lib.nb200_kv_attention(
        q.data_ptr(), packed, out.data_ptr(), batch, queries, heads, qb, qt, qh, ob, ot, oh,
        page_table.data_ptr(), page_table.stride(0), pages, lengths.data_ptr(),
        d ** -0.5 if scale is None else scale, window, sinks, code, _ptr(ws), need, stream))
    if given:
        increment_version(out)
    return out


def _logits(logits):
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError(f"'logits' must be [rows, vocabulary], got {tuple(shape)}")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"'logits' is {logits.dtype} (fp32, fp16 or bf16)")
    _rows("logits", logits, shape, logits.dtype)
    return shape


def _score(logits, tokens, top, inv_temperature, apart):
    """TokenLogprobs of checked arguments; `apart`: no two results in one tensor."""
    rows, vocab = logits.shape
    stream = _launch_stream("logits tokens", logits, tokens)
    if apart:
        logprob, entropy, lse = (logits.new_empty(rows, dtype=torch.float32) for _ in range(3))
    else:
        logprob, entropy, lse = logits.new_empty((3, rows), dtype=torch.float32).unbind(0)
    if tokens is None:
        logprob = None
    best = index = None
    if top:
        best = logits.new_empty((rows, top), dtype=torch.float32)
        index = logits.new_empty((rows, top), dtype=torch.int64)
    abi.check(abi.load().nb200_token_logprobs(
        logits.data_ptr(), _ptr(tokens), _ptr(logprob), entropy.data_ptr(), lse.data_ptr(),
        _ptr(best), _ptr(index), rows, vocab, logits.stride(0), top, inv_temperature,
        _CODES[logits.dtype], stream))
    return TokenLogprobs(logprob, entropy, lse, best, index)


class _RecordedScore(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, inv_temperature):
        got = _score(logits, tokens, top, inv_temperature, True)
        ctx.save_for_backward(logits, tokens, got.lse, got.entropy)
        ctx.inv_temperature = inv_temperature
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(got.top_index)
        return tuple(got)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, grad_lse, grad_top, _):
        if grad_lse is not None or grad_top is not None:
            raise NotImplementedError("token_logprobs has a gradient of logprob and entropy, not of lse and "
                                      "top_logprob: detach those")
        if grad_logprob is None and grad_entropy is None:
            return None, None, None, None
        logits, tokens, lse, entropy = ctx.saved_tensors
        # a sum's or a mean's gradient is one number for all rows
        dense = [g if g is None else g.contiguous() for g in (grad_logprob, grad_entropy)]
        return token_logprobs_backward(logits, tokens, lse, entropy, *dense,
                                       inv_temperature=ctx.inv_temperature), None, None, None


def token_logprobs(logits, tokens=None, top=0, inv_temperature=1.0):
    """Log probabilities of one given token per row of [rows, vocabulary] logits (fp32, fp16 or
    bf16), each row's entropy and log-sum-exp, and its `top` (up to 32) largest alternatives with
    their log probabilities, ties to the lower index.  tokens: int64 [rows]; a negative one stands
    for none and scores 0.  Returns TokenLogprobs of fp32 tensors (top_index: int64).

    Where gradients are enabled and the logits require one, logprob and entropy can be
    differentiated (once; the logits are kept until then); a gradient of lse or top_logprob is refused.
    A backward pass can be captured into a graph while no eager graph of the same leaves is alive, as
    any of torch's."""
    rows, vocab = _logits(logits)
    if tokens is not None:
        _vector("tokens", tokens, rows, torch.int64)
    if not 0 <= top <= 32:
        raise ValueError(f"token_logprobs: {top} alternatives (0 to 32)")
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_RecordedScore.apply(logits, tokens, top, inv_temperature))
    return _score(logits, tokens, top, inv_temperature, False)


def token_logprobs_backward(logits, tokens, lse, entropy, grad_logprob=None, grad_entropy=None,
                            inv_temperature=1.0, out=None):
    """The gradient of `token_logprobs` by its logits, in their type: of sum(grad_logprob * logprob)
    + sum(grad_entropy * entropy), with the lse and entropy that it returned.  `out` may be the
    logits themselves.  Not recorded for autograd: there is no second derivative."""
    rows, vocab = _logits(logits)
    if tokens is not None:
        _vector("tokens", tokens, rows, torch.int64)
    _vector("lse", lse, rows, torch.float32)
    _vector("entropy", entropy, rows, torch.float32)
    if grad_logprob is not None:
        _vector("grad_logprob", grad_logprob, rows, torch.float32)
    if grad_entropy is not None:
        _vector("grad_entropy", grad_entropy, rows, torch.float32)
    given = out is not None
    if given:
        _written("out", out, (rows, vocab), logits.dtype)
        if out is not logits:
            _no_backward("out", out)
    else:
        out = _fresh(logits, logits.dtype)
    stream = _launch_stream("logits tokens lse entropy grad_logprob grad_entropy out", logits, tokens,
                            lse, entropy, grad_logprob, grad_entropy, out)
    abi.check(abi.load().nb200_token_logprobs_bwd(
        logits.data_ptr(), _ptr(tokens), _ptr(lse), _ptr(entropy), _ptr(grad_logprob),
        _ptr(grad_entropy), out.data_ptr(), rows, vocab, logits.stride(0), out.stride(0),
        inv_temperature, _CODES[logits.dtype], stream))
    if given:
        increment_version(out)
    return out
