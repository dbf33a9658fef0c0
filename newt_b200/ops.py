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
nothing.  None of them records anything for autograd; `token_logprobs` has its gradient as a
function of its own.
"""

from typing import NamedTuple, Optional

import torch

from .runtime import abi

E4M3 = torch.float8_e4m3fn
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


def _shaped(name, t, shape, dtype=None):
    if t.shape != shape:
        raise ValueError(f"'{name}' has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"'{name}' is {t.dtype}, expected {dtype}")


def _dense_rows(name, t):
    """Rows may lie anywhere, the elements of a row side by side."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"'{name}' must have unit stride along its last dimension")


def _contiguous(name, t):
    if not t.is_contiguous():
        raise ValueError(f"'{name}' must be contiguous")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows_like(x, dtype):
    """A fresh contiguous tensor of x's shape."""
    if x.is_contiguous():
        return torch.empty_like(x, dtype=dtype)
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def rmsnorm(x, weight, residual=None, eps=1e-6, out_dtype=None, group=0, out=None, scales=None,
            residual_out=None):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight, over the rows of [rows, n] tensors
    (fp32, fp16 or bf16; n up to 32768).  Returns (out, scales, residual).

    `out_dtype` None: out = y in x's type.  torch.float8_e4m3fn: out = y / scale in 8 bits with
    scale = max|y| / 448 over the row (`group` 0; scales [rows, 1]) or over every `group` of 32, 64
    or 128 columns (scales [rows, ceil(n / group)]).  With a residual, h comes back in x's type.
    `out` and `residual_out` may be x and residual themselves."""
    if x.dim() != 2:
        raise ValueError(f"'x' must be [rows, n], got {tuple(x.shape)}")
    rows, n = x.shape
    dtype = x.dtype
    if out_dtype is None:
        out_dtype = dtype
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"rmsnorm: {dtype} (fp32, fp16 or bf16)")
    if out_dtype not in (dtype, E4M3):
        raise TypeError(f"rmsnorm: the output is {dtype} or float8_e4m3fn, not {out_dtype}")
    _shaped("weight", weight, (n,), dtype)
    _contiguous("weight", weight)
    if out is None:
        out = _rows_like(x, out_dtype)
    else:
        _shaped("out", out, (rows, n), out_dtype)
        _dense_rows("out", out)
    if out_dtype is E4M3:
        if group not in (0, 32, 64, 128):
            raise ValueError(f"rmsnorm: group {group} (0: one scale per row; 32, 64, 128 columns)")
        columns = -(-n // group) if group else 1
        if scales is None:
            scales = torch.empty((rows, columns), dtype=torch.float32, device=x.device)
        else:
            _shaped("scales", scales, (rows, columns), torch.float32)
            _dense_rows("scales", scales)
    elif group or scales is not None:
        raise ValueError("rmsnorm: scales and groups go with an e4m3 output")
    if residual is not None:
        _shaped("residual", residual, (rows, n), dtype)
        _dense_rows("residual", residual)
        if residual_out is None:
            residual_out = _rows_like(x, dtype)
        else:
            _shaped("residual_out", residual_out, (rows, n), dtype)
            _dense_rows("residual_out", residual_out)
    elif residual_out is not None:
        raise ValueError("rmsnorm: 'residual_out' goes with a residual")
    _dense_rows("x", x)
    stream = _launch_stream("x weight residual out scales residual_out", x, weight, residual, out,
                            scales, residual_out)
    abi.check(abi.load().nb200_rmsnorm(
        x.data_ptr(), _ptr(residual), weight.data_ptr(), out.data_ptr(), _ptr(residual_out),
        _ptr(scales), rows, n, x.stride(0), residual.stride(0) if residual is not None else 0,
        out.stride(0), residual_out.stride(0) if residual_out is not None else 0,
        scales.stride(0) if scales is not None else 0, group, eps, _CODES[dtype],
        _CODES[out_dtype], stream))
    return RmsNorm(out, scales, residual_out)


def _pack_cache(cache):
    """nb200_kv_cache of a KVCache, after its shapes and types have been looked at."""
    k, v, ks, vs = cache
    if k.dim() != 4:
        raise ValueError(f"'cache.k' must be [pages, heads, page_size, head_dim], got {tuple(k.shape)}")
    shape = k.shape
    pages, heads, page, d = shape
    if v.shape != shape:
        raise ValueError(f"'cache.v' has shape {tuple(v.shape)}, 'cache.k' {tuple(shape)}")
    if k.dtype is not E4M3 or v.dtype is not E4M3:
        raise TypeError(f"the cache holds {k.dtype} and {v.dtype}, expected float8_e4m3fn")
    _shaped("cache.k_scales", ks, (pages, heads), torch.float32)
    _shaped("cache.v_scales", vs, (pages, heads), torch.float32)
    kp, kh, kt, ku = k.stride()
    vp, vh, vt, vu = v.stride()
    if ku != 1 or vu != 1:
        raise ValueError("the cache must have unit stride along head_dim")
    ksp, ksh = ks.stride()
    vsp, vsh = vs.stride()
    if heads > 1 and (ksh != 1 or vsh != 1):
        raise ValueError("the cache's scales must have unit stride over heads")
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
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"'page_table' has shape {tuple(table.shape)}, expected ({batch}, pages)")
    if table.dtype is not torch.int32:
        raise TypeError(f"'page_table' is {table.dtype}, expected torch.int32")
    _dense_rows("page_table", table)


def kv_append(cache, k, v, page_table, starts, offsets, max_new):
    """Writes new keys and values into the cache, in place.

    k, v: [tokens, heads, head_dim] (fp16 or bf16), the new tokens of all sequences, one sequence
    after another; sequence b brings rows offsets[b] .. offsets[b + 1) (int32, [batch + 1]) and had
    starts[b] tokens before (int32).  page_table: int32 [batch, pages], the pages of each sequence
    in order.  max_new: at least the most new tokens of one sequence.

    Scales are powers of two, one per page and head; a page that holds older tokens keeps its scale
    or gets a larger one, to which the older tokens are then brought.  Sequences must not share the
    pages they write to.  Tokens whose page the table lacks are not written."""
    packed = _pack_cache(cache)
    pages, heads, page, d = cache.k.shape
    if k.dim() != 3 or k.shape[1:] != (heads, d):
        raise ValueError(f"'k' has shape {tuple(k.shape)}, expected (tokens, {heads}, {d})")
    _shaped("v", v, k.shape, k.dtype)
    if k.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"kv_append: {k.dtype} (fp16 or bf16)")
    _dense_rows("k", k)
    _dense_rows("v", v)
    batch = starts.shape[0]
    _shaped("starts", starts, (batch,), torch.int32)
    _shaped("offsets", offsets, (batch + 1,), torch.int32)
    _contiguous("starts", starts)
    _contiguous("offsets", offsets)
    _page_table(page_table, batch)
    stream = _launch_stream(
        "k v page_table starts offsets cache.k cache.v cache.k_scales cache.v_scales", k, v,
        page_table, starts, offsets, cache.k, cache.v, cache.k_scales, cache.v_scales)
    abi.check(abi.load().nb200_kv_append(
        packed, k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0), k.stride(1), v.stride(0),
        v.stride(1), page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
        starts.data_ptr(), offsets.data_ptr(), batch, max_new, _CODES[k.dtype], stream))


def kv_attention(q, cache, page_table, lengths, scale=None, window=0, sinks=0, out=None):
    """Attention of the newest tokens of each sequence over the cache.

    q: [batch, queries, heads, head_dim] (fp16 or bf16); heads is a multiple of the cache's heads.
    lengths: int32 [batch], the tokens of each sequence in the cache, the new ones among them: query
    i of sequence b stands at position lengths[b] - queries + i and sees the tokens up to its own,
    with `window` > 0 only the last `window` of them and the first `sinks` of the sequence.  A query
    that sees nothing gives zeros.  scale: 1 / sqrt(head_dim) if not given."""
    packed = _pack_cache(cache)
    if q.dim() != 4:
        raise ValueError(f"'q' must be [batch, queries, heads, head_dim], got {tuple(q.shape)}")
    batch, queries, heads, d = q.shape
    if d != cache.k.shape[3]:
        raise ValueError(f"'q' has head_dim {d}, the cache {cache.k.shape[3]}")
    dtype = q.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"kv_attention: {dtype} (fp16 or bf16)")
    _dense_rows("q", q)
    _shaped("lengths", lengths, (batch,), torch.int32)
    _contiguous("lengths", lengths)
    _page_table(page_table, batch)
    if out is None:
        out = _rows_like(q, dtype)
    else:
        _shaped("out", out, q.shape, dtype)
        _dense_rows("out", out)
    stream = _launch_stream(
        "q page_table lengths out cache.k cache.v cache.k_scales cache.v_scales", q, page_table,
        lengths, out, cache.k, cache.v, cache.k_scales, cache.v_scales)
    lib = abi.load()
    code = _CODES[dtype]
    need = lib.nb200_kv_attention_workspace_bytes(packed, batch, queries, heads, code)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    abi.check(lib.nb200_kv_attention(
        q.data_ptr(), packed, out.data_ptr(), batch, queries, heads, q.stride(0), q.stride(1),
        q.stride(2), out.stride(0), out.stride(1), out.stride(2), page_table.data_ptr(),
        page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
        d ** -0.5 if scale is None else scale, window, sinks, code, _ptr(ws), need, stream))
    return out


def _logits(logits):
    if logits.dim() != 2:
        raise ValueError(f"'logits' must be [rows, vocabulary], got {tuple(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"'logits' is {logits.dtype} (fp32, fp16 or bf16)")
    _dense_rows("logits", logits)
    return logits.shape


def _row_values(rows, dtype, **tensors):
    for name, t in tensors.items():
        if t is not None:
            _shaped(name, t, (rows,), dtype)
            _contiguous(name, t)


def token_logprobs(logits, tokens=None, top=0, inv_temperature=1.0):
    """Log probabilities of one given token per row of [rows, vocabulary] logits (fp32, fp16 or
    bf16), each row's entropy and log-sum-exp, and its `top` (up to 32) largest alternatives with
    their log probabilities, ties to the lower index.  tokens: int64 [rows]; a negative one stands
    for none and scores 0.  Returns TokenLogprobs of fp32 tensors (top_index: int64)."""
    rows, vocab = _logits(logits)
    _row_values(rows, torch.int64, tokens=tokens)
    if not 0 <= top <= 32:
        raise ValueError(f"token_logprobs: {top} alternatives (0 to 32)")
    stream = _launch_stream("logits tokens", logits, tokens)
    device = logits.device
    both = torch.empty((3, rows), dtype=torch.float32, device=device)
    logprob, entropy, lse = both.unbind(0)
    if tokens is None:
        logprob = None
    best = index = None
    if top:
        best = torch.empty((rows, top), dtype=torch.float32, device=device)
        index = torch.empty((rows, top), dtype=torch.int64, device=device)
    abi.check(abi.load().nb200_token_logprobs(
        logits.data_ptr(), _ptr(tokens), _ptr(logprob), entropy.data_ptr(), lse.data_ptr(),
        _ptr(best), _ptr(index), rows, vocab, logits.stride(0), top, inv_temperature,
        _CODES[logits.dtype], stream))
    return TokenLogprobs(logprob, entropy, lse, best, index)


def token_logprobs_backward(logits, tokens, lse, entropy, grad_logprob=None, grad_entropy=None,
                            inv_temperature=1.0, out=None):
    """The gradient of `token_logprobs` by its logits, in their type: of sum(grad_logprob * logprob)
    + sum(grad_entropy * entropy), with the lse and entropy that it returned.  `out` may be the
    logits themselves."""
    rows, vocab = _logits(logits)
    _row_values(rows, torch.int64, tokens=tokens)
    _row_values(rows, torch.float32, lse=lse, entropy=entropy, grad_logprob=grad_logprob,
                grad_entropy=grad_entropy)
    if out is None:
        out = _rows_like(logits, logits.dtype)
    else:
        _shaped("out", out, (rows, vocab), logits.dtype)
        _dense_rows("out", out)
    stream = _launch_stream("logits tokens lse entropy grad_logprob grad_entropy out", logits, tokens,
                            lse, entropy, grad_logprob, grad_entropy, out)
    abi.check(abi.load().nb200_token_logprobs_bwd(
        logits.data_ptr(), _ptr(tokens), _ptr(lse), _ptr(entropy), _ptr(grad_logprob),
        _ptr(grad_entropy), out.data_ptr(), rows, vocab, logits.stride(0), out.stride(0),
        inv_temperature, _CODES[logits.dtype], stream))
    return out
