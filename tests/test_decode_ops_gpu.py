"""The decode step's operators against plain implementations in 64 bits.

Tolerances: a result rounded to a type with relative step eps is off by at most eps / 2 of the
value.  What comes before that rounding is fp32 work; its part is written beside each test.
"""

import math

import pytest
import torch

from newt_b200 import examples, ops
from newt_b200.runtime import abi

pytestmark = pytest.mark.gpu

E4M3 = ops.E4M3
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF = {t: torch.finfo(t).eps / 2 for t in (BF16, FP16, FP32)}
TINY = {BF16: 1e-38, FP16: 2.0 ** -25, FP32: 1e-38}       # half a step among the subnormals


@pytest.fixture(autouse=True)
def _no_kernel_gave_up():
    yield
    torch.cuda.synchronize()
    assert abi.read_status() == (0, 0)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=FP32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _close(got, want, half, extra, floor):
    """|got - want| <= half a step of the value + what fp32 lost before the rounding."""
    got, want = got.double(), want.double()
    off = (got - want).abs() - ((half + extra) * want.abs() + floor)
    assert not torch.isnan(got).any() or torch.equal(torch.isnan(got), torch.isnan(want))
    worst = torch.nan_to_num(off, nan=0.0).max().item() if off.numel() else 0.0
    assert worst <= 0.0, worst


# ---- rmsnorm -----------------------------------------------------------------------------------

# y before its rounding: a sum of n squares in fp32 (pairwise over threads and lanes: at most 64
# additions deep, each off by 2^-24), a reciprocal root (2 ulp) and three products: below 2^-17.
RMS_EXTRA = 2.0 ** -17


def _rms_exact(x, w, residual, eps):
    h = x.double() + (residual.double() if residual is not None else 0.0)
    return h, h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def _check_rms(x, w, residual, got, out_dtype, group, eps):
    h, y = _rms_exact(x, w, residual, eps)
    dtype, n = x.dtype, x.shape[1]
    if residual is not None:
        # the fp32 sum of two numbers is off by 2^-24 of it before the rounding
        _close(got.residual, h, HALF[dtype], 2.0 ** -23, TINY[dtype])
    if out_dtype is not E4M3:
        _close(got.out, y, HALF[dtype], RMS_EXTRA, TINY[dtype])
        return
    width = group or n
    amax = torch.stack([part.abs().amax(1) for part in y.split(width, 1)], 1)
    scales = torch.where(amax > 0, amax / 448, 1.0)
    assert got.scales.shape == scales.shape
    _close(got.scales, scales, 0.0, RMS_EXTRA, 0.0)
    q = y / scales.repeat_interleave(width, 1)[:, :n]
    # half a step of e4m3 (2^-4 of the value, 2^-10 among the subnormals) and y's and the scale's
    # own errors, which also move a value across the middle between two numbers
    _close(got.out.float(), q, 2.0 ** -4, 4 * RMS_EXTRA, 2.0 ** -10 * 1.001)


@pytest.mark.parametrize("out, group", [(None, 0), (E4M3, 0), (E4M3, 32), (E4M3, 128)])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows, n", [(1, 1), (3, 8), (37, 100), (5, 257), (9, 1000), (2, 5003),
                                     (300, 4096), (3, 16384), (2, 32761), (2, 32768)])
def test_rmsnorm(rows, n, dtype, with_residual, out, group):
    gen = _gen(rows * 7 + n)
    x = _randn(gen, rows, n, dtype=dtype)
    residual = _randn(gen, rows, n, dtype=dtype, scale=3.0) if with_residual else None
    w = _randn(gen, n, dtype=dtype)
    got = ops.rmsnorm(x, w, residual=residual, eps=1e-5, out_dtype=out, group=group)
    _check_rms(x, w, residual, got, out, group, 1e-5)


def test_rmsnorm_of_strided_and_offset_rows():
    gen = _gen(3)
    wide = _randn(gen, 6, 700, dtype=BF16)
    w = _randn(gen, 256, dtype=BF16)
    for first in (0, 8, 3):             # rows on and off 16-byte boundaries
        x, residual = wide[:, first:first + 256], wide[:, 300 + first:556 + first]
        room = torch.full((6, 600), 7.0, device="cuda", dtype=BF16)
        out, res_out = room[:, first:first + 256], room[:, 300 + first:556 + first]
        got = ops.rmsnorm(x, w, residual=residual, eps=1e-6, out=out, residual_out=res_out)
        _check_rms(x, w, residual, got, None, 0, 1e-6)
        keep = torch.ones(600, dtype=torch.bool)
        keep[first:first + 256] = keep[300 + first:556 + first] = False
        assert (room[:, keep.cuda()] == 7.0).all()          # nothing beside the rows was written


@pytest.mark.parametrize("out, group", [(None, 0), (E4M3, 0), (E4M3, 32), (E4M3, 64), (E4M3, 128)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows, n", [(700, 5), (700, 129), (600, 1003), (400, 5122), (300, 16383)])
def test_rmsnorm_of_many_odd_rows(rows, n, dtype, out, group):
    """Rows that start at every remainder of 16 bytes, enough of them for several vectors per thread."""
    gen = _gen(rows + n)
    x, residual, w = (_randn(gen, *shape, dtype=dtype) for shape in ((rows, n), (rows, n), (n,)))
    got = ops.rmsnorm(x, w, residual=residual, eps=1e-5, out_dtype=out, group=group)
    _check_rms(x, w, residual, got, out, group, 1e-5)


@pytest.mark.parametrize("first", [1, 4, 7])
@pytest.mark.parametrize("n", [17, 256, 1001])
def test_rmsnorm_of_rows_that_start_alike(first, n):
    """All tensors off by the same remainder, and nothing beside their rows is written."""
    gen = _gen(first + n)
    x, residual = (_randn(gen, 9, n + 16, dtype=BF16)[:, first:first + n] for _ in range(2))
    w = _randn(gen, n, dtype=BF16)
    rooms = [torch.full((9, n + 16), 7.0, device="cuda", dtype=BF16) for _ in range(2)]
    codes = torch.full((9, n + 16), 0x55, device="cuda", dtype=torch.uint8)
    inside = [t[:, first:first + n] for t in rooms]
    got = ops.rmsnorm(x, w, residual=residual, eps=1e-5, out=inside[0], residual_out=inside[1])
    _check_rms(x, w, residual, got, None, 0, 1e-5)
    got = ops.rmsnorm(x, w, residual=residual, eps=1e-5, out_dtype=E4M3, group=32,
                      out=codes.view(E4M3)[:, first:first + n])
    _check_rms(x, w, residual, got, E4M3, 32, 1e-5)
    beside = torch.ones(n + 16, dtype=torch.bool, device="cuda")
    beside[first:first + n] = False
    assert (codes[:, beside] == 0x55).all() and all((t[:, beside] == 7.0).all() for t in rooms)


@pytest.mark.parametrize("n", [256, 4096, 1003])
def test_rmsnorm_over_its_own_inputs(n):
    gen = _gen(n)
    x, residual = _randn(gen, 500, n, dtype=BF16), _randn(gen, 500, n, dtype=BF16)
    w = _randn(gen, n, dtype=BF16)
    want = ops.rmsnorm(x, w, residual=residual)
    a, b = x.clone(), residual.clone()
    ops.rmsnorm(a, w, residual=b, out=a, residual_out=b)
    assert torch.equal(a, want.out) and torch.equal(b, want.residual)


def test_rmsnorm_of_zeros_and_of_what_is_not_finite():
    x = torch.zeros(4, 256, device="cuda", dtype=BF16)
    x[1, 5], x[2, 7], x[3] = float("nan"), float("inf"), 1e-30
    w = torch.ones(256, device="cuda", dtype=BF16)
    got = ops.rmsnorm(x, w, eps=0.5, out_dtype=E4M3, group=32)
    values = got.out.float() * got.scales.repeat_interleave(32, 1)
    assert (got.scales[0] == 1).all() and (values[0] == 0).all()
    assert torch.isnan(got.out.float()[1]).all()
    assert torch.isnan(got.out.float()[2, 7])
    assert torch.isfinite(got.scales[3]).all() and torch.isfinite(values[3]).all()
    assert (ops.rmsnorm(x[:1], w, eps=0.5).out == 0).all()
    none = ops.rmsnorm(x[:0], w, residual=x[:0])
    assert none.out.shape == (0, 256) and none.residual.shape == (0, 256)


# ---- the cache ---------------------------------------------------------------------------------

def _pages(gen, lengths, page, spare=2):
    """A page table in no order, -1 behind the last page of a sequence."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + spare
    ids = torch.randperm(total, generator=gen, device="cuda").tolist()
    table = torch.full((len(lengths), max(counts + [1]) + 1), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(ids[:c], dtype=torch.int32)
        ids = ids[c:]
    return table.cuda(), total


def _noise_cache(gen, pages, heads, page, d, order=(0, 1, 2, 3)):
    """Bytes of every kind, NaN among them, in a cache laid out in the given order of dimensions."""
    shape = (pages, heads, page, d)

    def tensor():
        laid = [shape[i] for i in order]
        t = torch.randint(0, 256, laid, generator=gen, device="cuda", dtype=torch.uint8)
        return t.permute([order.index(i) for i in range(4)]).view(E4M3)

    scales = [torch.exp2(torch.randint(-9, -4, (pages, heads), generator=gen,
                                       device="cuda").float()) for _ in range(2)]
    return ops.KVCache(tensor(), tensor(), *scales)


def _power(amax):
    m, e = math.frexp(amax)
    return 2.0 ** min(max(e - 9 if m <= 0.875 else e - 8, -60), 60) if amax > 0 else 2.0 ** -60


def _codes(values):
    """float64 values as e4m3 bytes, one rounding; NaN is 0x7F of its two bytes."""
    codes = values.clamp(-448, 448).float().to(E4M3).view(torch.uint8)
    codes[values.isnan()] = 0x7F
    return codes


def _append_plain(cache, k, v, table, starts, offsets):
    """What kv_append is defined to leave, token by token and page by page, on the CPU."""
    out = []
    for x, codes, scales in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
        x, scales = x.cpu().double(), scales.cpu().clone()
        codes = codes.view(torch.uint8).cpu().clone()
        page, heads = codes.shape[2], codes.shape[1]
        for b, start in enumerate(starts.tolist()):
            low, high = offsets[b].item(), offsets[b + 1].item()
            end = start + high - low
            for at in range(start // page, -(-end // page)):
                if at >= table.shape[1] or not 0 <= table[b, at].item() < codes.shape[0]:
                    continue
                where = table[b, at].item()
                first, last = max(start - at * page, 0), min(end - at * page, page)
                for h in range(heads):
                    rows = x[low + at * page + first - start:low + at * page + last - start, h]
                    finite = rows[~rows.isnan()]
                    need = _power(finite.abs().max().item() if finite.numel() else 0.0)
                    if first:
                        before = scales[where, h].item()
                        need = max(need, before)
                        if need > before:
                            old = codes[where, h, :first].view(E4M3).double() * (before / need)
                            codes[where, h, :first] = _codes(old)
                    codes[where, h, first:last] = _codes(rows / need)
                    scales[where, h] = need
        out.append((codes, scales))
    return out


def _check_append(cache, k, v, table, starts, offsets, most):
    want = _append_plain(cache, k, v, table.cpu(), starts.cpu(), offsets.cpu())
    for again in range(2):              # the second call finds its own result
        ops.kv_append(cache, k, v, table, starts, offsets, most)
        for codes, scales, (want_codes, want_scales) in ((cache.k, cache.k_scales, want[0]),
                                                         (cache.v, cache.v_scales, want[1])):
            # scales are exact, and so is a value over a power of two: one rounding, the same one
            assert torch.equal(scales.cpu(), want_scales)
            assert torch.equal(codes.view(torch.uint8).cpu(), want_codes)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (0, 2, 1, 3), (1, 0, 2, 3)])
@pytest.mark.parametrize("page, d, heads, dtype", [(16, 64, 3, FP16), (16, 128, 1, BF16),
                                                   (32, 128, 2, FP16), (64, 64, 8, BF16),
                                                   (128, 128, 2, BF16), (128, 64, 1, FP16)])
def test_append(page, d, heads, dtype, order):
    gen = _gen(page + d)
    starts = [0, 5, page, page - 1, 3 * page - 2, 17, 0]
    new = [1, 3, 2 * page, 1, page + 5, 0, 1]
    table, total = _pages(gen, [a + b for a, b in zip(starts, new)], page)
    cache = _noise_cache(gen, total, heads, page, d, order)
    offsets = [sum(new[:i]) for i in range(len(new) + 1)]
    rows = offsets[-1] + 3                       # three rows of padding behind the last sequence
    k, v = (_randn(gen, rows, heads, d, dtype=dtype, scale=s) for s in (4.0, 0.01))
    k[2] *= 100.0                                # one page whose scale has to grow
    k[offsets[-1]:] = float("inf")
    _check_append(cache, k, v, table, _int32(starts), _int32(offsets), max(new))


def test_append_of_rows_that_are_not_aligned_or_lie_apart():
    gen = _gen(5)
    table, total = _pages(gen, [40, 9], 16)
    wide = _randn(gen, 30, 4, 150, dtype=BF16)
    for first in (0, 8, 1):
        cache = _noise_cache(gen, total, 2, 16, 64)
        k, v = wide[:, ::2, first:first + 64], wide[:, 1:3, 70 + first:134 + first]
        _check_append(cache, k, v, table, _int32([19, 0]), _int32([0, 21, 30]), 21)


def test_append_skips_pages_that_are_not_there():
    gen = _gen(6)
    cache = _noise_cache(gen, 4, 2, 16, 64)
    before = [t.clone() for t in cache]
    k = _randn(gen, 64, 2, 64, dtype=BF16)
    for table, starts in (([[-1, 4]], [0]), ([[1 << 30, -7]], [0]), ([[0, 1]], [32]), ([[0, 1]], [-5]),
                          ([[0, 1]], [2 ** 31 - 1])):
        ops.kv_append(cache, k, k, _int32(table), _int32(starts), _int32([0, 32]), 32)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(cache, before))
    # offsets beyond the rows there are, and backwards ones, bring nothing from outside
    ops.kv_append(cache, k[:8], k[:8], _int32([[0, 1]]), _int32([0]), _int32([9, 40]), 32)
    ops.kv_append(cache, k[:8], k[:8], _int32([[0, 1]]), _int32([0]), _int32([5, 2]), 32)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    # half of a sequence's pages there
    _check_append(cache, k, k, _int32([[2, -1, 3]]), _int32([3]), _int32([0, 40]), 40)


def test_append_of_extreme_values():
    gen = _gen(7)
    cache = _noise_cache(gen, 6, 1, 16, 64)
    x = torch.zeros(6 * 16, 1, 64, device="cuda", dtype=BF16)
    x[16:32] = 3e38                        # beyond 448 * 2^60: the largest value
    x[32:48] = 1e-38                       # below 2^-60 of anything: zero
    x[48:64] = 448.0
    x[64:80] = 449.0                       # in bf16, whose steps are 2 here, 448 again
    x[80:96, 0, 3], x[80:96, 0, 4] = float("nan"), 7.0
    _check_append(cache, x, -x, _int32([[0, 1, 2, 3, 4, 5]]), _int32([0]), _int32([0, 96]), 96)
    assert cache.k_scales[:, 0].tolist() == [2.0 ** -60, 2.0 ** 60, 2.0 ** -60, 1.0, 1.0, 2.0 ** -6]
    assert torch.isnan(cache.k.float()[5, 0, :, 3]).all()
    _check_append(cache, x[:16] + 450, x[:16], _int32([[0]]), _int32([0]), _int32([0, 16]), 16)
    assert cache.k_scales[0, 0] == 2.0     # the next scale


# ---- attention over the cache ------------------------------------------------------------------

def _attend_exact(q, cache, table, lengths, scale, window, sinks):
    """(out, mean magnitude of the visible values), from the definition, in 64 bits."""
    batch, nq, heads, d = q.shape
    kv_heads, page = cache.k.shape[1], cache.k.shape[2]
    out = torch.zeros(batch, nq, heads, d, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    for b, length in enumerate(lengths.tolist()):
        j = torch.arange(min(max(length, 0), table.shape[1] * page), device="cuda")
        ids = table[b].long()[j // page]
        there = (ids >= 0) & (ids < cache.k.shape[0])
        ids = ids.clamp(0, cache.k.shape[0] - 1)
        def tokens(codes, scales):
            got = codes.view(torch.uint8)[ids, :, j % page].view(E4M3).to(torch.float64)
            return (got * scales.double()[ids][:, :, None]).repeat_interleave(heads // kv_heads, 1)
        k, v = tokens(cache.k, cache.k_scales), tokens(cache.v, cache.v_scales)
        for i in range(nq):
            at = length - nq + i
            seen = there & (j <= at)
            if window:
                seen &= (j > at - window) | (j < sinks)
            if not seen.any():
                continue
            s = torch.einsum("hd,jhd->hj", q[b, i].double(), k[seen]) * scale
            p = torch.softmax(s, 1)
            out[b, i] = torch.einsum("hj,jhd->hd", p, v[seen])
            size[b, i] = torch.einsum("hj,jhd->hd", p, v[seen].abs())
    return out, size


def _check_attention(got, q, cache, table, lengths, scale=None, window=0, sinks=0):
    d = q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    want, size = _attend_exact(q, cache, table, lengths, scale, window, sinks)
    # Before the last rounding, relative to the mean magnitude of the values seen:
    # - a probability in [1, 2) times a power of two is rounded to fp16: half a step is 2^-11.  For
    #   bf16 two e4m3 parts hold it: the first leaves up to half its step, 2^-4, and the second up to
    #   half the step of a number below 2^-4, which is 2^-9.  For fp16 three parts of 4 bits hold the
    #   11 bits exactly.
    # - a score is an fp32 sum of d products, off by at most d 2^-24 sum |q k| scale < 2^-11 for the
    #   inputs below, and so is its exponential;
    # - a probability below 2^-22 of its 256 tokens' largest may be lost: 256 of them are 2^-14.
    extra = {BF16: 2.0 ** -9 + 2.0 ** -11, FP16: 2.0 ** -11}[q.dtype] + 2.0 ** -11 + 2.0 ** -14
    off = (got.double() - want).abs() - (HALF[q.dtype] * want.abs() + extra * size + TINY[q.dtype])
    assert not torch.isnan(off).any()
    assert off.max().item() <= 0.0, off.max().item()


def _finite_cache(gen, pages, heads, page, d, order=(0, 1, 2, 3)):
    cache = _noise_cache(gen, pages, heads, page, d, order)
    for t in (cache.k, cache.v):
        codes = t.view(torch.uint8)
        codes[(codes & 127) > 0x60] = 0x30       # values up to 32: scores of a few units
    return cache


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 300, 1000]


@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (40, 3), (128, 0), (200, 130), (5000, 4)])
@pytest.mark.parametrize("page, d, heads, kv_heads, nq, dtype", [
    (16, 64, 3, 3, 1, FP16), (16, 128, 8, 1, 1, BF16), (32, 128, 14, 2, 2, BF16),
    (64, 64, 8, 2, 3, FP16), (64, 128, 32, 8, 1, FP16), (128, 128, 8, 2, 8, BF16),
    (128, 64, 2, 2, 5, BF16), (16, 64, 40, 1, 3, BF16), (32, 128, 24, 1, 4, FP16)])
def test_attention(page, d, heads, kv_heads, nq, dtype, window, sinks):
    gen = _gen(page + d + nq)
    table, total = _pages(gen, LENGTHS, page)
    cache = _finite_cache(gen, total, kv_heads, page, d)
    q = _randn(gen, len(LENGTHS), nq, heads, d, dtype=dtype)
    lengths = _int32(LENGTHS)
    got = ops.kv_attention(q, cache, table, lengths, window=window, sinks=sinks)
    _check_attention(got, q, cache, table, lengths, window=window, sinks=sinks)


@pytest.mark.parametrize("order", [(0, 2, 1, 3), (1, 0, 2, 3)])
def test_attention_of_other_layouts_and_strides(order):
    gen = _gen(21)
    lengths = _int32([70, 333])
    table, total = _pages(gen, [70, 333], 32)
    cache = _finite_cache(gen, total, 2, 32, 64, order)
    wide = _randn(gen, 2, 6, 3, 80, dtype=BF16)
    q = wide.transpose(1, 2)[:, :, :4, 5:69]          # [2, 3, 4, 64] off a 16-byte boundary
    room = torch.full((2, 4, 3, 70), 7.0, device="cuda", dtype=BF16)
    out = room.transpose(1, 2)[..., 3:67]
    assert ops.kv_attention(q, cache, table, lengths, scale=0.3, out=out) is out
    _check_attention(out, q, cache, table, lengths, scale=0.3)
    assert (room[..., :3] == 7.0).all() and (room[..., 67:] == 7.0).all()


@pytest.mark.parametrize("page, d", [(16, 128), (64, 64), (128, 128)])
def test_attention_does_not_look_at_what_no_query_sees(page, d):
    """NaN in every byte that no query of the call sees: behind the last token, before the window,
    in pages of others, in the scales of pages that are not read."""
    gen = _gen(31)
    for length, window, sinks in ((37, 0, 0), (129, 0, 0), (700, 50, 4), (1000, 130, 1), (0, 0, 0)):
        table, total = _pages(gen, [length, 3], page)
        cache = _finite_cache(gen, total, 2, page, d)
        j = torch.arange(length, device="cuda")
        seen = (j > length - 1 - window) | (j < sinks) if window else j >= 0
        keep = torch.zeros(total, page, dtype=torch.bool, device="cuda")
        keep[table[0].long()[j[seen] // page], j[seen] % page] = True
        for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
            codes.view(torch.uint8).transpose(1, 2)[~keep] = 0x7F
            scales[~keep.any(1)] = float("nan")
        q = _randn(gen, 1, 1, 4, d, dtype=BF16)
        lengths = _int32([length])
        got = ops.kv_attention(q, cache, table[:1], lengths, window=window, sinks=sinks)
        _check_attention(got, q, cache, table[:1], lengths, window=window, sinks=sinks)


def test_attention_of_pages_that_are_not_there():
    gen = _gen(41)
    cache = _finite_cache(gen, 6, 2, 16, 128)
    q = _randn(gen, 4, 2, 4, 128, dtype=BF16)
    table = _int32([[0, -1, 2], [-1, -1, -1], [6, 1 << 30, 3], [4, 5, 1]])
    for lengths in ([48, 48, 48, 48], [40, 3, 17, 100], [-1, -2 ** 31, 2 ** 31 - 1, 1]):
        lengths = _int32(lengths)
        got = ops.kv_attention(q, cache, table, lengths)
        _check_attention(got, q, cache, table, lengths)


def test_attention_of_scales_far_apart():
    """Pages whose scales differ by up to 2^75: the small values' part must not vanish, the large ones'
    must not overflow."""
    gen = _gen(51)
    cache = _finite_cache(gen, 16, 1, 16, 64)
    cache.k_scales.fill_(2.0 ** -6)
    cache.v_scales[:] = torch.exp2(torch.arange(16, device="cuda").float() * 5 - 40)[:, None]
    q = _randn(gen, 1, 1, 2, 64, dtype=BF16, scale=0.5)
    table = torch.randperm(16, generator=gen, device="cuda").int()[None]
    for length in (256, 130, 16):
        lengths = _int32([length])
        _check_attention(ops.kv_attention(q, cache, table, lengths), q, cache, table, lengths)


def test_attention_of_scores_far_apart():
    """Scores of hundreds, of both signs: one token takes everything."""
    gen = _gen(52)
    table, total = _pages(gen, [900], 64)
    cache = _finite_cache(gen, total, 1, 64, 128)
    q = _randn(gen, 1, 1, 8, 128, dtype=BF16, scale=40.0)
    lengths = _int32([900])
    got = ops.kv_attention(q, cache, table, lengths)
    want, size = _attend_exact(q, cache, table, lengths, 128 ** -0.5, 0, 0)
    # scores of up to 2^11: fp32 has them to 2^-12, sums of 128 products to 2^-9 or so
    off = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -5 * size)
    assert off.max() <= 0
    zero = ops.kv_attention(torch.zeros_like(q), cache, table, lengths)
    _check_attention(zero, torch.zeros_like(q), cache, table, lengths)


def test_attention_beyond_32_bit_offsets():
    """A cache of 5 GB (keys and values in one tensor), its last pages in use."""
    gen = _gen(61)
    pages, heads = 40000, 8
    codes = torch.zeros(pages, heads, 128, 128, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.full((pages, heads), 2.0 ** -5, device="cuda")
    cache = ops.KVCache(codes, codes, scales, scales)
    table = _int32([[pages - 1, 1, pages - 3, pages // 2]])
    k = _randn(gen, 500, heads, 128, dtype=BF16)
    ops.kv_append(cache, k, k, table, _int32([0]), _int32([0, 500]), 500)
    assert codes[pages - 1].float().abs().max() > 0
    small = ops.KVCache(codes[table[0].long()], codes[table[0].long()], scales[table[0].long()],
                        scales[table[0].long()])
    q = _randn(gen, 1, 1, 16, 128, dtype=BF16)
    got = ops.kv_attention(q, cache, table, _int32([500]))
    _check_attention(got, q, small, _int32([[0, 1, 2, 3]]), _int32([500]))


def test_attention_of_a_long_sequence_and_many_short_ones():
    gen = _gen(62)
    lengths = [20011] + [33] * 200
    table, total = _pages(gen, lengths, 32)
    cache = _finite_cache(gen, total, 2, 32, 64)
    q = _randn(gen, 201, 1, 4, 64, dtype=BF16)
    lengths = _int32(lengths)
    first = ops.kv_attention(q, cache, table, lengths)
    _check_attention(first, q, cache, table, lengths)
    for _ in range(3):                           # the same bits every time
        assert torch.equal(ops.kv_attention(q, cache, table, lengths), first)


# ---- log probabilities -------------------------------------------------------------------------

def _score_exact(x, tokens, inv):
    z = x.double() * inv
    top = z.amax(1, keepdim=True)       # first: 3e38 + 8 is 3e38 in 64 bits too
    log_sum = (z - top).exp().sum(1, keepdim=True).log()
    lse = (top + log_sum)[:, 0]
    log_p = z - top - log_sum
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    picked = log_p.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    return torch.where(tokens < 0, 0.0, picked), entropy, lse, log_p


def _check_scores(x, tokens, top, inv, got=None):
    got = ops.token_logprobs(x, tokens, top=top, inv_temperature=inv) if got is None else got
    logprob, entropy, lse, log_p = _score_exact(x, tokens, inv)
    # fp32: a logit minus the maximum, times 1/T, is off by 2^-23 of its size (below 2^8 here, so
    # 2^-15 at the largest, which only has weight where it is small); the sum of a row by less than
    # 2^-20 of itself, the logarithm with it; the entropy by that times the size of the logits.
    for mine, want in ((got.logprob, logprob), (got.entropy, entropy), (got.lse, lse)):
        _close(mine, want, HALF[FP32], 2.0 ** -21, 2.0 ** -18)
    if not top:
        assert got.top_index is None and got.top_logprob is None
        return
    order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(got.top_index, order)
    _close(got.top_logprob, log_p.gather(1, order), HALF[FP32], 2.0 ** -21, 2.0 ** -18)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (37, 1000), (2, 4099),
                                         (1, 129001), (300, 5001), (700, 8192)])
def test_token_logprobs(rows, vocab, dtype):
    gen = _gen(rows + vocab)
    x = _randn(gen, rows, vocab, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    for top, inv in ((0, 1.0), (1, 0.7), (min(20, vocab), 1.0), (min(32, vocab), 2.0)):
        _check_scores(x, tokens, top, inv)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_token_logprobs_of_ordered_and_equal_logits(vocab, dtype):
    """Every order that fills the candidates' list, and rows of nothing but ties."""
    up = torch.linspace(-4, 4, vocab, device="cuda")
    gen = _gen(vocab)
    few = torch.randint(0, 3, (vocab,), generator=gen, device="cuda").float()
    signed = torch.where(few > 1, 0.0, -0.0) * torch.ones(vocab, device="cuda")
    x = torch.stack([up, up.flip(0), torch.zeros_like(up), few, signed,
                     up.view(-1)[torch.randperm(vocab, generator=gen, device="cuda")],
                     torch.sin(up * 50)]).to(dtype)
    tokens = torch.zeros(7, dtype=torch.int64, device="cuda")
    for top in (1, 7, 32):
        _check_scores(x, tokens, top, 1.0)
    many = x.repeat(100, 1)                       # one CTA per row
    _check_scores(many, tokens.repeat(100), 20, 1.0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_token_logprobs_of_masked_logits(dtype):
    gen = _gen(71)
    vocab, low, inf = 3001, torch.finfo(dtype).min, float("inf")
    x = _randn(gen, 6, vocab, dtype=dtype, scale=2.0)
    x[0, 5:] = -inf                               # five tokens left
    x[1, :2999] = low
    x[2] = low                                    # all alike: uniform
    x[3] = -inf
    x[3, 1234] = 2.0                              # one token left
    x[4, ::2] = torch.finfo(dtype).max            # half of them far above
    tokens = torch.tensor([3, 5, 7, 1234, 2, -100], device="cuda")
    got = ops.token_logprobs(x, tokens, top=6, inv_temperature=1.0)
    logprob, entropy, lse, log_p = _score_exact(x, tokens, 1.0)
    for mine, want in ((got.logprob, logprob), (got.entropy, entropy), (got.lse, lse)):
        finite = torch.isfinite(want.float())
        assert torch.equal(mine[~finite].double(), want[~finite])
        _close(mine[finite], want[finite], HALF[FP32], 2.0 ** -21, 2.0 ** -18)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :6]
    assert torch.equal(got.top_index, order)
    assert got.logprob[5] == 0
    ones = torch.ones(6, device="cuda")
    grad = ops.token_logprobs_backward(x, tokens, got.lse, got.entropy, ones, ones)
    assert torch.isfinite(grad).all()
    if dtype is not FP16:
        assert (grad[2] == 0).all()               # masked as a whole


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("vocab", [3, 100, 1023, 4099, 20011])
def test_token_logprobs_of_many_rows(vocab, dtype):
    """More rows than the chip has SMs: each is one small CTA's."""
    gen = _gen(vocab)
    x = _randn(gen, 301, vocab, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, vocab, (301,), generator=gen, device="cuda")
    for top, inv in ((0, 1.0), (1, 0.7), (min(5, vocab), 1.25), (min(32, vocab), 2.0)):
        _check_scores(x, tokens, top, inv)


@pytest.mark.parametrize("rows, vocab, dtype", [(150, 30011, BF16), (296, 16384, FP16), (297, 20005, BF16),
                                               (500, 17003, FP16), (593, 16390, BF16), (400, 9001, FP32)])
def test_token_logprobs_of_rows_that_share_the_chip(rows, vocab, dtype):
    """Around once, twice and four times as many rows as SMs, long enough for two small CTAs each."""
    gen = _gen(rows)
    x = _randn(gen, rows, vocab, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    for top in (0, 5, 32):
        _check_scores(x, tokens, top, 1.0)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [3, 200, 400])
@pytest.mark.parametrize("vocab", [33, 1000, 4099, 20000])
def test_alternatives_of_any_order(vocab, rows, dtype):
    """Equal, ordered, sparse and bunched logits: no list overflows and ties go to the lower index."""
    gen = _gen(vocab + rows)
    steps = torch.arange(vocab, device="cuda").float() * (20.0 / vocab)
    sparse = torch.full((vocab,), -math.inf, device="cuda")
    sparse[::max(1, vocab // 9)] = 1.0
    bunched = _randn(gen, vocab)
    bunched[::8] += 50.0
    not_numbers = _randn(gen, vocab)
    not_numbers[::7] = math.nan
    lowest = torch.full((vocab,), torch.finfo(dtype).min, device="cuda")
    for row in (torch.full((vocab,), 1.5, device="cuda"), steps, -steps, steps.round(), sparse, bunched,
                not_numbers, lowest, sparse - math.inf):
        x = row.to(dtype).expand(rows, vocab).contiguous()
        order = torch.sort(x.float().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=1,
                           descending=True, stable=True)[1]
        for top in (1, 2, 7, 32):
            assert torch.equal(ops.token_logprobs(x, top=top).top_index, order[:, :top])


def test_token_logprobs_of_rows_without_any_and_of_nan():
    x = torch.full((4, 5000), float("-inf"), device="cuda")
    x[1, 77], x[1, 78] = float("nan"), 1.0
    x[2, 3], x[2, 4] = float("inf"), 1.0
    x[3] = 0.0
    tokens = torch.tensor([0, 78, 4, 5000], device="cuda")
    got = ops.token_logprobs(x, tokens, top=3)
    assert got.logprob[0] == -math.inf and got.lse[0] == -math.inf and got.entropy[0] == 0
    assert got.top_index[0].tolist() == [0, 1, 2] and (got.top_logprob[0] == -math.inf).all()
    assert all(torch.isnan(t[1:3]).all() for t in (got.logprob, got.entropy, got.lse))
    assert got.top_index[2, 0] == 3
    assert torch.isnan(got.logprob[3])            # a token beyond the vocabulary
    grad = ops.token_logprobs_backward(x, tokens, got.lse, got.entropy,
                                       torch.ones(4, device="cuda"), torch.ones(4, device="cuda"))
    assert (grad[0] == 0).all() and torch.isnan(grad[1]).any()
    assert torch.isfinite(grad[3]).all()


def test_token_logprobs_of_strided_rows_and_without_tokens():
    gen = _gen(81)
    wide = _randn(gen, 20, 2100, dtype=BF16)
    tokens = torch.randint(0, 1003, (10,), generator=gen, device="cuda")
    for first in range(0, 9):
        x = wide[::2, first:first + 1003]
        got = ops.token_logprobs(x, tokens, top=4)
        _check_scores(x, tokens, 4, 1.0, got)
        bare = ops.token_logprobs(x)
        assert bare.logprob is None and torch.equal(bare.lse, got.lse)
        assert torch.equal(bare.entropy, got.entropy)
    assert ops.token_logprobs(wide[:0], tokens[:0], top=3).top_index.shape == (0, 3)


def _grad_exact(x, tokens, g, ge, inv):
    logprob, entropy, lse, log_p = _score_exact(x, tokens, inv)
    p = log_p.exp()
    g = torch.where((tokens >= 0) & (tokens < x.shape[1]), g.double(), 0.0)
    hit = torch.zeros_like(p).scatter_(1, tokens.clamp(0, x.shape[1] - 1)[:, None], 1.0)
    d = g[:, None] * (hit - p)
    inner = torch.where(p > 0, log_p, 0.0) + entropy[:, None]
    return inv * (d - ge.double()[:, None] * p * inner)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows, vocab, inv", [(1, 1, 1.0), (3, 7, 0.5), (65, 1000, 1.0),
                                              (5, 4099, 2.0), (2, 129001, 1.0), (300, 50, 1.0)])
def test_token_logprobs_backward(rows, vocab, inv, dtype):
    gen = _gen(rows * 3 + vocab)
    x = _randn(gen, rows, vocab, dtype=dtype, scale=2.0)
    if vocab > 100:
        x[:, -20:] = float("-inf")
    tokens = torch.randint(0, max(1, vocab - 20), (rows,), generator=gen, device="cuda")
    tokens[::3] = -100
    if rows > 1:
        tokens[1] = vocab
    g, ge = _randn(gen, rows), _randn(gen, rows, scale=0.3)
    f = ops.token_logprobs(x, tokens, inv_temperature=inv)
    want = _grad_exact(x, tokens, g, ge, inv)
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, g, ge, inv_temperature=inv)
    # p is off by the error of its exponent, below 2^-19 for exponents up to 2^5; the bracket it is
    # multiplied with by 2^-20 of the sizes that cancel in it
    p = (x.double() * inv - f.lse.double()[:, None]).exp()
    size = p * (g.abs()[:, None] + ge.abs()[:, None] * 32) * inv
    off = (got.double() - want).abs() - (HALF[dtype] * want.abs() + 2.0 ** -18 * size + TINY[dtype])
    off -= (tokens[:, None] == torch.arange(vocab, device="cuda")) * (g.abs()[:, None] * inv * 2.0 ** -22)
    assert off.max() <= 0, off.max()
    only = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, g, inv_temperature=inv)
    zero = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, g, torch.zeros_like(ge),
                                       inv_temperature=inv)
    assert torch.equal(only, zero)
    over = x.clone()
    ops.token_logprobs_backward(over, tokens, f.lse, f.entropy, g, ge, inv_temperature=inv, out=over)
    assert torch.equal(over, got)


def test_token_logprobs_backward_against_differences():
    """d f / d x_j by central differences of the forward pass in fp32, of a small vocabulary: the
    forward's error of 2^-20 over a step of 2 * 2^-5 allows 2^-15, the third derivative's part
    (2^-5)^2 / 6 of a few units 2^-11."""
    gen = _gen(91)
    x = _randn(gen, 1, 40, scale=1.5)
    tokens = torch.tensor([7], device="cuda")
    f = ops.token_logprobs(x, tokens, inv_temperature=0.8)
    got = ops.token_logprobs_backward(x, tokens, f.lse, f.entropy, torch.full((1,), 1.5, device="cuda"),
                                      torch.full((1,), -0.5, device="cuda"), inv_temperature=0.8)
    step = 2.0 ** -5
    shift = torch.eye(40, device="cuda") * step

    def value(z):
        r = ops.token_logprobs(z, tokens.expand(40).contiguous(), inv_temperature=0.8)
        return 1.5 * r.logprob.double() - 0.5 * r.entropy.double()

    slope = (value(x + shift) - value(x - shift)) / (2 * step)
    assert (slope - got[0].double()).abs().max() <= 2.0 ** -10


# ---- streams, graphs, together -----------------------------------------------------------------

def _step_inputs(gen, dtype=BF16):
    lengths = [130, 1, 47]
    table, total = _pages(gen, [n + 4 for n in lengths], 16)
    cache = _finite_cache(gen, total, 2, 16, 64)
    x = _randn(gen, 3, 256, dtype=dtype)
    k, v = _randn(gen, 3, 2, 64, dtype=dtype), _randn(gen, 3, 2, 64, dtype=dtype)
    q = _randn(gen, 3, 1, 8, 64, dtype=dtype)
    logits = _randn(gen, 3, 5003, dtype=dtype)
    return lengths, table, cache, x, k, v, q, logits


def _step(lengths, table, cache, x, k, v, q, logits, w, offsets, tokens):
    h = ops.rmsnorm(x, w, residual=x, out_dtype=E4M3, group=64)
    ops.kv_append(cache, k, v, table, lengths, offsets, 1)
    o = ops.kv_attention(q, cache, table, lengths + 1, window=100, sinks=2)
    s = ops.token_logprobs(logits, tokens, top=5)
    d = ops.token_logprobs_backward(logits, tokens, s.lse, s.entropy, s.logprob, s.entropy)
    return [h.out.float(), h.scales, h.residual, o, d, *s]


def test_the_operators_in_a_graph_and_on_another_stream():
    gen = _gen(101)
    lengths, table, cache, x, k, v, q, logits = _step_inputs(gen)
    w = _randn(gen, 256, dtype=BF16)
    offsets, tokens = _int32([0, 1, 2, 3]), torch.tensor([1, 2, 3], device="cuda")
    at = _int32(lengths)
    start = [t.clone() for t in cache]
    args = (at, table, cache, x, k, v, q, logits, w, offsets, tokens)

    def fresh():
        for t, s in zip(cache, start):
            t.view(torch.uint8).copy_(s.view(torch.uint8)) if t.dtype == E4M3 else t.copy_(s)

    want = [t.clone() for t in _step(*args)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fresh_done = torch.cuda.Event()
    fresh()
    fresh_done.record()
    side.wait_event(fresh_done)
    with torch.cuda.stream(side):
        got = _step(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    graphs = []
    for _ in range(2):                           # two graphs, replayed one after the other
        fresh()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = _step(*args)
        graphs.append((g, got))
    for g, got in graphs:
        fresh()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the same graph with other lengths, queries and logits in its inputs
    fresh()
    at.copy_(_int32([131, 2, 48]))
    q.copy_(_randn(gen, 3, 1, 8, 64, dtype=BF16))
    logits.copy_(_randn(gen, 3, 5003, dtype=BF16))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    after = [t.clone() for t in graphs[0][1]]
    fresh()
    assert all(torch.equal(a, b) for a, b in zip(after, _step(*args)))


def test_two_steps_at_once():
    """The same operators on two streams, nothing but their inputs in common, with sequences long
    enough that the attention's parts are joined."""
    gen = _gen(131)
    lengths = [5000, 1, 2300]
    table, total = _pages(gen, [n + 1 for n in lengths], 16)
    x = _randn(gen, 3, 1003, dtype=BF16)
    w = _randn(gen, 1003, dtype=BF16)
    k, v = _randn(gen, 3, 2, 64, dtype=BF16), _randn(gen, 3, 2, 64, dtype=BF16)
    q = _randn(gen, 3, 1, 8, 64, dtype=BF16)
    logits = _randn(gen, 3, 50021, dtype=BF16)
    offsets, tokens, at = _int32([0, 1, 2, 3]), torch.tensor([1, 2, 3], device="cuda"), _int32(lengths)
    first = _finite_cache(gen, total, 2, 16, 64)
    caches = [ops.KVCache(*(t.clone() for t in first)) for _ in range(3)]
    args = lambda i: (at, table, caches[i], x, k, v, q, logits, w, offsets, tokens)
    want = _step(*args(2))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):                          # the append may be repeated
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = _step(*args(i))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_with_nothing_to_do():
    gen = _gen(17)
    cache = _finite_cache(gen, 4, 2, 16, 64)
    before = [t.clone() for t in cache]
    q = _randn(gen, 2, 3, 4, 64, dtype=FP16)
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    table = _int32([[0, 1], [2, 3]])
    # no table, no tokens: nothing is seen
    assert (ops.kv_attention(q, cache, none, _int32([40, 0])) == 0).all()
    assert (ops.kv_attention(q, cache, table, _int32([0, -3])) == 0).all()
    assert ops.kv_attention(q[:0], cache, table[:0], _int32([])).shape == (0, 3, 4, 64)
    k = _randn(gen, 5, 2, 64, dtype=FP16)
    ops.kv_append(cache, k, k, none, _int32([0, 0]), _int32([0, 2, 5]), 3)
    ops.kv_append(cache, k, k, table, _int32([0, 0]), _int32([0, 0, 0]), 3)
    ops.kv_append(cache, k[:0], k[:0], table, _int32([0, 0]), _int32([0, 0, 0]), 3)
    for t, was in zip(cache, before):
        assert torch.equal(*((a.view(torch.uint8) if a.dtype == E4M3 else a) for a in (t, was)))
    # a bound on the new tokens that is far too large costs nothing and changes nothing
    _check_append(cache, k, k, table, _int32([0, 3]), _int32([0, 2, 5]), 2 ** 31 - 1)


def test_a_prompt_and_its_decode_steps():
    """One layer of a decoder, prompt first and then token by token, on the framework's own
    product and the operators here, against the whole sequence at once in 64 bits."""
    gen = _gen(111)
    dtype, d, heads, kv_heads, hidden, vocab = BF16, 64, 8, 2, 256, 1000
    w_norm = (1 + 0.1 * _randn(gen, hidden)).to(dtype)
    w_qkv = _randn(gen, hidden, (heads + 2 * kv_heads) * d, dtype=dtype, scale=hidden ** -0.5)
    w_out = _randn(gen, heads * d, vocab, dtype=dtype, scale=0.3)
    total, prompt, window, sinks = 150, 141, 60, 3
    x = _randn(gen, total, hidden, dtype=dtype)
    cache = ops.new_kv_cache(16, kv_heads, 16, d)
    table = torch.randperm(16, generator=gen, device="cuda").int()[None]
    outs, scores = [], []
    done = 0
    for new in [prompt] + [1] * (total - prompt):
        y = ops.rmsnorm(x[done:done + new], w_norm).out
        qkv = examples.matmul(y, w_qkv).view(new, heads + 2 * kv_heads, d)
        ops.kv_append(cache, qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], table,
                      _int32([done]), _int32([0, new]), new)
        done += new
        o = ops.kv_attention(qkv[None, :, :heads], cache, table, _int32([done]), window=window,
                             sinks=sinks)[0]
        logits = examples.matmul(o.reshape(new, heads * d), w_out)
        outs.append(o)
        scores.append(ops.token_logprobs(logits, torch.arange(done - new, done, device="cuda")))
    got = torch.cat(outs).double()

    y = (x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * w_norm.double())
    qkv = (y @ w_qkv.double()).view(total, -1, d)
    k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in
            (qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]))
    s = torch.einsum("ihd,jhd->hij", qkv[:, :heads], k) * d ** -0.5
    i, j = torch.arange(total, device="cuda")[:, None], torch.arange(total, device="cuda")
    seen = (j <= i) & ((j > i - window) | (j < sinks))
    p = torch.softmax(s.masked_fill(~seen, -math.inf), 2)
    want = torch.einsum("hij,jhd->ihd", p, v)
    # keys and values in e4m3 are off by up to 2^-4 of themselves, 2^-5 / sqrt(3) in the mean: of the
    # same order in the output, far below the 1 that unrelated numbers would be off
    assert ((got - want).norm() / want.norm()).item() < 0.08
    log_p = torch.log_softmax(want.reshape(total, -1) @ w_out.double(), 1)
    mine = torch.cat([t.logprob for t in scores]).double()
    picked = log_p[torch.arange(total), torch.arange(total)]
    assert (mine - picked).abs().mean().item() < 0.1


def test_attention_of_many_sequences_of_few_tiles():
    """More sequences than shares of the work, of one to four steps each: shares of whole items, and
    a table so short that no workspace is asked for."""
    gen = _gen(63)
    for longest in (700, 1000):
        lengths = [1 + (i * 37) % longest for i in range(311)]
        lengths[5] = longest
        table, total = _pages(gen, lengths, 64)
        table = table[:, :-(-longest // 64)].contiguous()
        cache = _finite_cache(gen, total, 1, 64, 64)
        q = _randn(gen, 311, 1, 2, 64, dtype=BF16)
        lengths = _int32(lengths)
        _check_attention(ops.kv_attention(q, cache, table, lengths), q, cache, table, lengths)
