"""GPU: the serving operators against their 64-bit definitions (serving_reference.py).

Tolerances.  With u half a step of the type (2^-11 fp16, 2^-8 bf16), one output element is
off by at most u A for the rounding of the probabilities (A = sum p |v|), u |o| for the store,
2 ds A for scores that are off by ds, and a few fp32 roundings (2^-18 A covers the sums and
the exponentials' 2^-22); fp16 probabilities under 2^-14 round absolutely, by 2^-25 each.
ds: an fp32 sum of d products is off by at most d 2^-24 sum |q k| scale.  The log-sum-exp is
off by ds and a few roundings of its own size."""
import math

import pytest
import torch

from serving_reference import (attention_block, attention_rows, cache_rows, evict_choice,
                               lengths_to_offsets)
from tttj_2026_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(out, lse, q, k, v, n, length, scale, causal=True, rows=False):
    """One sequence: out / lse [n, H, ...] of its last n of `length` tokens."""
    f = attention_rows if rows else attention_block
    ref, ref_lse = f(q, k, v, n, length, scale, causal)
    d, u = q.shape[2], torch.finfo(q.dtype).eps / 2
    g = q.shape[1] // k.shape[1]
    qn = torch.nan_to_num(q.double().abs()).amax((0, 1)) if n else torch.zeros(d, device=DEV, dtype=torch.float64)
    kn = torch.nan_to_num(k.double().abs(), posinf=0).amax((0, 1))
    ds = d * 2.0**-24 * float((qn * kn).sum()) * scale
    vabs = torch.nan_to_num(v.double().abs(), posinf=0)
    a, _ = f(q, torch.nan_to_num(k, posinf=0, neginf=0), vabs.to(v.dtype), n, length, scale, causal)
    tol = (u + 2 * ds + 2.0**-18) * a + u * ref.abs() + (2.0**-25 * (1 + vabs.sum(0)).repeat_interleave(g, 0)
                                                          if q.dtype == torch.float16 else 0)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(out.double()), torch.isnan(ref))
    assert torch.equal(torch.isposinf(out.double()), torch.isposinf(ref))
    assert torch.equal(torch.isneginf(out.double()), torch.isneginf(ref))
    err = (out.double() - ref).abs()
    assert bool((err <= tol)[fin].all()), f"out: {float((err / tol)[fin].max()):.2f} times the tolerance"
    lfin = torch.isfinite(ref_lse)
    assert torch.equal(torch.isneginf(lse.double()), torch.isneginf(ref_lse))
    lerr = (lse.double() - ref_lse).abs()[lfin]
    ltol = (ds + 2.0**-20 * (1 + ref_lse.abs()))[lfin]
    assert bool((lerr <= ltol).all()), f"lse: {float((lerr / ltol).max()):.2f} times the tolerance"


# ------------------------------------------------------------------------------- prompts
def _prompt(lens, heads, kv, d, dtype, seed, spread=1.5):
    t = sum(lens)
    qkv = torch.randn(t, (heads + 2 * kv) * d, device=DEV, generator=_gen(seed)).to(dtype)
    q, k, v = qkv.split((heads * d, kv * d, kv * d), 1)
    q.mul_(spread)
    return q.view(t, heads, d), k.view(t, kv, d), v.view(t, kv, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (8, 1), (5, 1)])
@pytest.mark.parametrize("lens", [[1], [77, 0, 200, 1, 129], [513, 2, 255]])
def test_prompt_attention(dtype, d, heads, kv, lens):
    q, k, v = _prompt(lens, heads, kv, d, dtype, sum(lens) + d)
    off = lengths_to_offsets(lens)
    for causal in (True, False):
        out, lse = ops.prompt_attention(q, k, v, off, causal=causal, return_lse=True)
        at = 0
        for n in lens:
            s = slice(at, at + n)
            if n:
                _check(out[s], lse[s], q[s], k[s], v[s], n, n, d**-0.5, causal)
            at += n


@pytest.mark.parametrize("group", [7, 16, 33, 64])
def test_prompt_attention_wide_groups(group):
    lens = [3, 150, 40]
    q, k, v = _prompt(lens, 2 * group, 2, 64, torch.float16, group)
    out, lse = ops.prompt_attention(q, k, v, lengths_to_offsets(lens), return_lse=True, scale=0.2)
    at = 0
    for n in lens:
        s = slice(at, at + n)
        _check(out[s], lse[s], q[s], k[s], v[s], n, n, 0.2)
        at += n


def test_prompt_attention_long_and_sharp():
    """A long prompt whose scores reach far: running maxima that keep growing."""
    q, k, v = _prompt([2500], 4, 2, 128, torch.bfloat16, 5, spread=8.0)
    k.mul_(torch.linspace(0.2, 2, 2500, device=DEV)[:, None, None])
    out, lse = ops.prompt_attention(q, k, v, lengths_to_offsets([2500]), return_lse=True)
    _check(out, lse, q, k, v, 2500, 2500, 128**-0.5)


def test_prompt_attention_rows_behind_the_last_sequence_stay():
    q, k, v = _prompt([40, 30, 58], 4, 2, 64, torch.float16, 3)
    k[70:], v[70:], q[70:] = math.nan, math.inf, math.nan
    out = torch.full((128, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    got = ops.prompt_attention(q, k, v, lengths_to_offsets([40, 30]), out=out)
    assert got is out
    assert bool((out[70:] == 7).all())
    for s in (slice(0, 40), slice(40, 70)):
        ref, _ = attention_block(q[s], k[s], v[s], s.stop - s.start, s.stop - s.start, 64**-0.5)
        assert float((out[s].double() - ref).abs().max()) < 0.01


def test_prompt_attention_strided_rows():
    base = torch.randn(90, 3, 5, 96, device=DEV, generator=_gen(1)).half()
    q, k, v = base[:, 0, :4, 8:72], base[:, 1, 1:3, 16:80], base[:, 2, ::2, 32:][:, :2]
    big = torch.zeros(90, 8, 72, dtype=torch.float16, device=DEV)
    out = ops.prompt_attention(q, k, v, lengths_to_offsets([33, 57]), out=big[:, ::2, 8:])
    for s in (slice(0, 33), slice(33, 90)):
        n = s.stop - s.start
        lse = attention_block(q[s], k[s], v[s], n, n, 0.125)[1]
        _check(out[s], lse, q[s], k[s], v[s], n, n, 0.125)
    assert bool((big[:, 1::2] == 0).all()) and bool((big[:, :, :8] == 0).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_attention_nonfinite_values_reach_only_rows_that_see_them(d, dtype):
    lens = [140, 9, 300]
    q, k, v = _prompt(lens, 4, 2, d, dtype, 11)
    v[37, 0, 3], v[100, 1, 5], v[101, 1, 5] = math.nan, math.inf, -math.inf
    v[145, 0, 0] = -math.inf
    k[148, 1] = math.nan  # the last token of the second sequence: only its own row sees it
    v[149 + 200, 1, d - 1] = math.inf
    out, lse = ops.prompt_attention(q, k, v, lengths_to_offsets(lens), return_lse=True)
    at = 0
    for n in lens:
        s = slice(at, at + n)
        _check(out[s], lse[s], q[s], k[s], v[s], n, n, d**-0.5, rows=True)
        at += n


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_attention_a_channel_of_nan_values(d):
    """Every row sees a NaN in one channel, and hides others: that channel is NaN, no other is."""
    q, k, v = _prompt([1500], 4, 2, d, torch.float16, 12)
    v[:, 1, 5] = math.nan
    out, lse = ops.prompt_attention(q, k, v, lengths_to_offsets([1500]), return_lse=True)
    assert bool(torch.isnan(out[:, 2:, 5]).all())
    v[:, 1, 5], out[:, 2:, 5] = 0, 0
    _check(out, lse, q, k, v, 1500, 1500, d**-0.5)


# -------------------------------------------------------------------------- paged cache
class Cache:
    def __init__(self, lens, kv, d, page, dtype, seed, spare=5, heads_first=False, extra_pages=0):
        b = len(lens)
        self.per = max(1, -(-max(lens) // page)) + extra_pages
        pages = b * self.per + spare
        shape = (pages, kv, page, d) if heads_first else (pages, page, kv, d)
        g = _gen(seed)
        self.k = torch.full(shape, math.nan, dtype=dtype, device=DEV)
        self.v = torch.full(shape, math.inf, dtype=dtype, device=DEV)
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(pages, generator=g, device=DEV)[: b * self.per]
        self.table = order.to(torch.int32).view(b, self.per).contiguous()
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        for i, n in enumerate(lens):  # only live slots hold finite values
            j = torch.arange(n, device=DEV)
            at = self.table[i].long()[j // page]
            self.k[at, j % page] = torch.randn(n, kv, d, device=DEV, generator=g).to(dtype)
            self.v[at, j % page] = torch.randn(n, kv, d, device=DEV, generator=g).to(dtype)


def _check_cache(out, lse, q, c, new, lens, scale, rows=False):
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        if n:
            s = slice(at, at + n)
            if m == 0:
                assert bool((out[s] == 0).all()) and bool(torch.isneginf(lse[s]).all())
            else:
                _check(out[s], lse[s], q[s], cache_rows(c.k, c.table, b, m), cache_rows(c.v, c.table, b, m), n, m,
                       scale, rows=rows or m < n)
        at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv", [(8, 2), (3, 3), (10, 2)])
def test_cache_attention_single_tokens(dtype, d, page, heads, kv):
    lens = [1, 15, 16, 17, 63, 64, 65, 300, 129, 1000]
    c = Cache(lens, kv, d, page, dtype, d + page)
    q = (1.5 * torch.randn(len(lens), heads, d, device=DEV, generator=_gen(2))).to(dtype)
    new = [1] * len(lens)
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, max_new=1, return_lse=True)
    _check_cache(out, lse, q, c, new, lens, d**-0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv,page", [(8, 2, 16), (3, 3, 32), (10, 2, 128), (16, 1, 64)])
def test_cache_attention_chunks(dtype, d, heads, kv, page):
    new = [5, 0, 1, 130, 33, 64]
    lens = [5, 40, 700, 130, 500, 257]
    c = Cache(lens, kv, d, page, dtype, d + page)
    q = (1.5 * torch.randn(sum(new), heads, d, device=DEV, generator=_gen(2))).to(dtype)
    for hint in (None, max(new), 1):
        out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, max_new=hint,
                                       return_lse=True)
        _check_cache(out, lse, q, c, new, lens, d**-0.5)


@pytest.mark.parametrize("new", [1, 3, 200])
def test_cache_attention_long_axis_is_split(new):
    """One sequence, many keys: the work of its few rows is shared between CTAs and joined."""
    lens = [20011]
    c = Cache(lens, 2, 128, 64, torch.bfloat16, 4)
    q = (2 * torch.randn(new, 8, 128, device=DEV, generator=_gen(5))).bfloat16()
    args = (q, c.k, c.v, c.table, lengths_to_offsets([new]), c.lens)
    out, lse = ops.cache_attention(*args, max_new=new, return_lse=True)
    _check_cache(out, lse, q, c, [new], lens, 128**-0.5)
    again = ops.cache_attention(*args, max_new=new)
    assert torch.equal(out, again)  # joined in a fixed order


def test_cache_attention_heads_first_pages():
    new, lens = [1, 40, 1], [90, 333, 64]
    c = Cache(lens, 3, 64, 32, torch.float16, 8, heads_first=True)
    q = torch.randn(sum(new), 6, 64, device=DEV, generator=_gen(5)).half()
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, return_lse=True)
    _check_cache(out, lse, q, c, new, lens, 0.125)


def test_cache_attention_rows_that_see_nothing():
    """More new tokens than cached ones: the first of them see no key; an empty cache."""
    new, lens = [4, 3, 70], [2, 0, 69]
    c = Cache(lens, 2, 64, 16, torch.float16, 8)
    q = torch.randn(sum(new), 4, 64, device=DEV, generator=_gen(5)).half()
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, return_lse=True)
    assert bool((out[:2] == 0).all()) and bool(torch.isneginf(lse[:2]).all())
    assert bool((out[7] == 0).all()) and bool(torch.isneginf(lse[7]).all())
    _check_cache(out, lse, q, c, new, lens, 0.125)


@pytest.mark.parametrize("new", [[3, 1], [60, 50]])
def test_cache_attention_nonfinite_values_reach_only_rows_that_see_them(new):
    lens = [131, 80]
    c = Cache(lens, 2, 128, 16, torch.bfloat16, 8)
    j = 129  # seen by the last two new tokens of the first sequence only
    c.v[c.table[0, j // 16].long(), j % 16, 1, 77] = math.nan
    c.v[c.table[0, (j + 1) // 16].long(), (j + 1) % 16, 0, 3] = -math.inf
    c.k[c.table[1, 79 // 16].long(), 79 % 16, 0] = math.nan
    q = torch.randn(sum(new), 4, 128, device=DEV, generator=_gen(5)).bfloat16()
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, return_lse=True)
    _check_cache(out, lse, q, c, new, lens, 128**-0.5, rows=True)


@pytest.mark.parametrize("new", [3, 150])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_cache_attention_nonfinite_values_in_split_keys(d, new):
    """As above where one sequence's keys are shared out between CTAs: hidden values in the last
    part, one that every row sees in the first."""
    lens = [9001]
    c = Cache(lens, 2, d, 64, torch.float16, 8)
    for j, h, x in ((8999, 0, math.nan), (9000, 1, math.inf)):
        c.v[c.table[0, j // 64].long(), j % 64, h, 5] = x
    c.v[c.table[0, 1].long(), 3, 1, 7] = -math.inf
    q = torch.randn(new, 8, d, device=DEV, generator=_gen(5)).half()
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets([new]), c.lens, return_lse=True)
    _check_cache(out, lse, q, c, [new], lens, d**-0.5, rows=True)


def test_cache_attention_wrong_pages_and_lengths_are_contained():
    """Page numbers outside the cache stand for zeros, lengths for the table's slots."""
    lens = [100, 64, 30]
    c = Cache(lens, 2, 64, 16, torch.float16, 8)
    c.table[0, 2] = -7
    c.table[1, 1] = 1 << 30
    q = torch.randn(3, 4, 64, device=DEV, generator=_gen(5)).half()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    off = lengths_to_offsets([1, 1, 1])
    out = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, status=status)
    assert int(status) == 0x401
    for b, (bad, m) in enumerate([(2, 100), (1, 64), (None, 30)]):
        table = c.table.clone().clamp_(0, c.k.shape[0] - 1)
        k, v = cache_rows(c.k, table, b, m).clone(), cache_rows(c.v, table, b, m).clone()
        if bad is not None:
            k[bad * 16:(bad + 1) * 16], v[bad * 16:(bad + 1) * 16] = 0, 0
        ref, _ = attention_block(q[b:b + 1], k, v, 1, m, 0.125)
        assert float((out[b] - ref).abs().max()) < 0.01
    status.zero_()
    c = Cache([112, 64, 30], 2, 64, 16, torch.float16, 8)
    lens = torch.tensor([1 << 30, 64, -5], dtype=torch.int32, device=DEV)
    out = ops.cache_attention(q, c.k, c.v, c.table, off, lens, status=status)
    assert int(status) == 0x402
    ref, _ = attention_block(q[:1], cache_rows(c.k, c.table, 0, 112), cache_rows(c.v, c.table, 0, 112), 1, 112, 0.125)
    assert float((out[0] - ref).abs().max()) < 0.01
    assert bool((out[2] == 0).all())
    status.zero_()
    bad_off = torch.tensor([-3, 1, 90, 3], dtype=torch.int32, device=DEV)
    ops.cache_attention(q, c.k, c.v, c.table, bad_off, c.lens, status=status)
    assert int(status) == 0x402


@pytest.mark.parametrize("new", [1, 100])
def test_cache_attention_behind_2_31_elements(new):
    """Pages whose elements lie beyond 32-bit offsets."""
    pages, page, kv, d = 70000, 64, 4, 128
    k = torch.empty(pages, page, kv, d, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    c = Cache([150], kv, d, page, torch.float16, 3)
    table = torch.tensor([[69999, 66001, 65537]], dtype=torch.int32, device=DEV)
    k[table[0].long()], v[table[0].long()] = c.k[c.table[0].long()], c.v[c.table[0].long()]
    q = torch.randn(new, 8, d, device=DEV, generator=_gen(5)).half()
    out, lse = ops.cache_attention(q, k, v, table, lengths_to_offsets([new]), c.lens, return_lse=True)
    _check_cache(out, lse, q, c, [new], [150], d**-0.5)
    nk = torch.randn(new, kv, d, device=DEV, generator=_gen(6)).half()
    ops.cache_append(nk, nk + 1, k, v, table, lengths_to_offsets([new]), c.lens)
    c.k, c.v, c.table = k, v, table
    assert torch.equal(cache_rows(k, table, 0, 150)[150 - new:], nk)
    assert torch.equal(cache_rows(v, table, 0, 150)[150 - new:], nk + 1)


def test_captured_calls_follow_new_lengths():
    """One graph of append + attention, replayed with other lengths, pages and tokens."""
    kv, heads, d, page = 2, 8, 64, 16
    c = Cache([200, 200, 200], kv, d, page, torch.float16, 3)
    off = lengths_to_offsets([1, 1, 1])
    q = torch.zeros(3, heads, d, dtype=torch.float16, device=DEV)
    nk, nv = torch.zeros(3, kv, d, dtype=torch.float16, device=DEV), torch.zeros(3, kv, d, dtype=torch.float16, device=DEV)

    def step():
        ops.cache_append(nk, nv, c.k, c.v, c.table, off, c.lens)
        return ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=1, return_lse=True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i, lens in enumerate([[3, 77, 200], [1, 16, 17], [100, 0, 64]]):
        g = _gen(20 + i)
        q.copy_(torch.randn(q.shape, device=DEV, generator=g))
        nk.copy_(torch.randn(nk.shape, device=DEV, generator=g))
        nv.copy_(torch.randn(nk.shape, device=DEV, generator=g))
        c.lens.copy_(torch.tensor(lens))
        c.table.copy_(c.table.flatten()[torch.randperm(c.table.numel(), device=DEV, generator=g)].view_as(c.table))
        c.k.copy_(torch.randn(c.k.shape, device=DEV, generator=g))
        c.v.copy_(torch.randn(c.v.shape, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for b, m in enumerate(lens):
            if m:
                assert torch.equal(cache_rows(c.k, c.table, b, m)[-1], nk[b])
        _check_cache(out, lse, q, c, [1, 1, 1], lens, 0.125)


def test_serving_on_another_stream():
    lens = [100, 300]
    c = Cache(lens, 2, 64, 16, torch.float16, 3)
    q = torch.randn(2, 4, 64, device=DEV, generator=_gen(5)).half()
    off = lengths_to_offsets([1, 1])
    want = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.cache_attention(q, c.k, c.v, c.table, off, c.lens) for _ in range(20)]
    side.synchronize()
    assert all(torch.equal(want, g) for g in got)


# -------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,kv", [(32, 16, 3), (64, 64, 1), (128, 32, 8), (256, 256, 2)])
def test_cache_append(dtype, d, page, kv):
    new, lens = [1, 0, 17, 300, 5], [1, 9, 40, 300, 3]
    c = Cache([300] * 5, kv, d, page, dtype, 3, extra_pages=1)
    c.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k0, v0 = c.k.clone(), c.v.clone()
    rows = torch.randn(sum(new) + 4, 2 * kv + 1, d, device=DEV, generator=_gen(1)).to(dtype)
    k, v = rows[:, :kv], rows[:, kv:2 * kv]
    cap = c.table.shape[1] * page
    pos = torch.full((5, kv, cap), 77, dtype=torch.int32, device=DEV)
    mass = torch.full((5, kv, cap), 5.0, device=DEV)
    seen = torch.tensor([11, 12, 1000, 300, 1 << 20], dtype=torch.int32, device=DEV)
    ops.cache_append(k, v, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, positions=pos, mass=mass, seen=seen)
    at = 0
    want_pos, want_mass = torch.full_like(pos, 77), torch.full_like(mass, 5.0)
    for b, (n, m) in enumerate(zip(new, lens)):
        skip = max(0, n - m)  # tokens before the cache's first slot are dropped
        for i in range(skip, n):
            slot = m - n + i
            page_at = int(c.table[b, slot // page])
            k0[page_at, slot % page], v0[page_at, slot % page] = k[at + i], v[at + i]
            want_pos[b, :, slot], want_mass[b, :, slot] = int(seen[b]) - n + i, 0
        at += n
    # compared as bits: most of the cache is NaN here
    assert torch.equal(c.k.contiguous().view(torch.int16), k0.contiguous().view(torch.int16))
    assert torch.equal(c.v.contiguous().view(torch.int16), v0.contiguous().view(torch.int16))
    assert torch.equal(pos, want_pos) and torch.equal(mass, want_mass)


def test_cache_append_drops_tokens_of_wrong_pages():
    c = Cache([64, 64], 2, 64, 16, torch.float16, 3)
    k0 = c.k.clone()
    c.table[0, 3] = 10**6
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = torch.randn(3, 2, 64, device=DEV, generator=_gen(1)).half()
    ops.cache_append(k, k, c.k, c.v, c.table, lengths_to_offsets([1, 2]), c.lens, status=status)
    assert int(status) == 0x401
    at = c.table[1, 3].long()
    k0[at, 14], k0[at, 15] = k[1], k[2]
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))


# ----------------------------------------------------------------------------- eviction
def _evict_case(lens, kv, d, page, dtype, seed, heads_first=False):
    c = Cache(lens, kv, d, page, dtype, seed, heads_first=heads_first)
    b, cap = len(lens), c.table.shape[1] * page
    g = _gen(seed + 1)
    mass = torch.exp(torch.randn(b, kv, cap, device=DEV, generator=g))
    mass = (mass * 8).round() / 8  # many equal ones
    pos = torch.rand(b, kv, cap, device=DEV, generator=g).argsort(2).to(torch.int32)
    return c, mass, pos


def _check_evict(c, mass, pos, lens, keep, recent):
    k0, v0 = c.k.clone(), c.v.clone()
    page = c.k.shape[1]
    got_mass, got_pos, got_lens = ops.cache_evict(mass, pos, c.k, c.v, c.table, c.lens, keep, recent=recent)
    want_mass, want_pos = mass.clone(), pos.clone()
    for b, m in enumerate(lens):
        t = c.table[b].long()
        for h in range(c.k.shape[2]):
            hole, mover = evict_choice(mass[b, h], pos[b, h], m, keep, recent)
            assert len(hole) == len(mover)
            if hole:
                hole, mover = torch.tensor(hole, device=DEV), torch.tensor(mover, device=DEV)
                for cache in (k0, v0):
                    cache[t[hole // page], hole % page, h] = cache[t[mover // page], mover % page, h]
                want_mass[b, h, hole], want_pos[b, h, hole] = mass[b, h, mover], pos[b, h, mover]
        want_mass[b, :, min(m, keep):], want_pos[b, :, min(m, keep):] = 0, -1
    assert got_lens.tolist() == [min(m, keep) for m in lens]
    assert torch.equal(got_pos, want_pos)
    assert torch.equal(got_mass.view(torch.int32), want_mass.view(torch.int32))
    assert torch.equal(c.k.contiguous().view(torch.int16), k0.contiguous().view(torch.int16))
    assert torch.equal(c.v.contiguous().view(torch.int16), v0.contiguous().view(torch.int16))
    return got_mass, got_pos, got_lens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,kv", [(32, 16, 3), (64, 64, 1), (128, 32, 2), (256, 128, 2)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (100, 30), (64, 64), (511, 0), (5000, 9)])
def test_cache_evict(dtype, d, page, kv, keep, recent):
    lens = [0, 1, 64, 100, 101, 700, 512]
    c, mass, pos = _evict_case(lens, kv, d, page, dtype, 9)
    _check_evict(c, mass, pos, lens, keep, recent)


def test_cache_evict_special_masses():
    """NaN, infinities, both zeros, negative numbers, denormals, all equal."""
    lens = [300, 300, 200]
    c, mass, pos = _evict_case(lens, 2, 64, 16, torch.float16, 9, heads_first=True)
    odd = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0, 1e-42, -1e-42, 3e38], device=DEV)
    mass[0] = odd[torch.randint(0, 9, mass[0].shape, device=DEV, generator=_gen(1))]
    mass[1] = 0.25
    _check_evict(c, mass, pos, lens, 128, 16)


@pytest.mark.parametrize("keep", [99, 100, 101, 159, 160, 161])
def test_cache_evict_cut_beside_zero(keep):
    """100 positive masses, 60 zeros of either sign, 40 negative ones, in any order."""
    lens = [200, 200]
    c, mass, pos = _evict_case(lens, 2, 64, 16, torch.float16, 9)
    g = _gen(4)
    for b in range(2):
        for h in range(2):
            row = torch.rand(200, device=DEV, generator=g) + 0.1
            row[100:160] = torch.where(torch.rand(60, device=DEV, generator=g) < 0.5, 0.0, -0.0)
            row[160:] *= -1
            mass[b, h, :200] = row[torch.randperm(200, device=DEV, generator=g)]
    _check_evict(c, mass, pos, lens, keep, 0)


@pytest.mark.parametrize("length", [40000, 70000])
def test_cache_evict_long(length):
    """Longer than what the selection holds in shared memory, and just below."""
    lens = [length, 30000]
    c, mass, pos = _evict_case(lens, 1, 32, 256, torch.float16, 9)
    _check_evict(c, mass, pos, lens, 8000, 100)


# -------------------------------------------------------------------------- gathered mass
def _check_mass(got, mass, q, lse, c, new, lens, scale):
    """Each probability is off by its score's error ds (see above), the log-sum-exp's
    rounding in the log2 domain (2^-23 of its size) and the exponential's 2^-22; sums of m
    terms by m 2^-24 relative, taken as one."""
    d = q.shape[2]
    at = 0
    want, tol = mass.double(), torch.zeros_like(mass, dtype=torch.float64)
    for b, (n, m) in enumerate(zip(new, lens)):
        if n and m:
            k = cache_rows(c.k, c.table, b, m)
            g = q.shape[1] // k.shape[1]
            s = torch.einsum("nhd,mhd->hnm", q[at:at + n].double(), k.double().repeat_interleave(g, 1)) * scale
            sa = torch.einsum("nhd,mhd->hnm", q[at:at + n].double().abs(), k.double().abs().repeat_interleave(g, 1))
            hidden = torch.ones(n, m, dtype=torch.bool, device=DEV).triu(m - n + 1)
            w = torch.exp(s - lse[at:at + n].double().t()[:, :, None]).masked_fill(hidden, 0)
            e = w * (d * 2.0**-24 * sa * scale + 2.0**-21 * (1 + s.abs() + lse[at:at + n].double().t().abs()[:, :, None]))
            want[b, :, :m] += w.view(k.shape[1], -1, m).sum(1)
            tol[b, :, :m] += e.view(k.shape[1], -1, m).sum(1)
        at += n
    tol += (sum(new) * q.shape[1] + 2) * 2.0**-24 * want.abs()
    err = (got.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), f"{float((err / (tol + 1e-30)).max()):.2f} times the tolerance"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv,page", [(8, 2, 16), (3, 3, 32), (10, 2, 128), (16, 1, 256), (6, 2, 64)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1, 1, 1], [1, 16, 127, 129, 1000]),
                                      ([5, 0, 1, 130, 33, 300], [5, 40, 700, 130, 500, 301])])
def test_cache_mass(dtype, d, heads, kv, page, new, lens):
    c = Cache(lens, kv, d, page, dtype, d + page)
    q = (1.5 * torch.randn(sum(new), heads, d, device=DEV, generator=_gen(2))).to(dtype)
    off, scale = lengths_to_offsets(new), d**-0.5
    mass = torch.rand(len(lens), kv, c.table.shape[1] * page, device=DEV, generator=_gen(3))
    _, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=max(new), return_lse=True)
    for hint in (None, max(new), 1):
        got = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass, max_new=hint)
        _check_mass(got, mass, q, lse, c, new, lens, scale)
    again = mass.clone()
    assert ops.cache_mass(q, lse, c.k, c.table, off, c.lens, again, max_new=max(new), out=again) is again
    assert torch.equal(again, ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass, max_new=max(new)))


def test_cache_mass_hidden_and_empty():
    """Rows that see nothing, padded rows, NaN keys and queries that others do not see."""
    new, lens = [4, 3, 70, 2], [2, 0, 69, 40]
    c = Cache(lens, 2, 64, 16, torch.float16, 8)
    q = torch.randn(sum(new) + 5, 4, 64, device=DEV, generator=_gen(5)).half()
    off = lengths_to_offsets(new)
    _, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, return_lse=True)
    lse[sum(new):] = math.nan
    q[sum(new):] = math.nan
    mass = torch.rand(4, 2, c.table.shape[1] * 16, device=DEV, generator=_gen(3))
    got = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass)
    want = mass.double()
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        for i in range(n):
            see = max(0, m - n + i + 1)
            k = cache_rows(c.k, c.table, b, m)[:see].double()
            for h in range(4):
                s = k[:, h // 2] @ q[at + i, h].double() * 0.125
                want[b, h // 2, :see] += torch.exp(s - lse[at + i, h].double())
        at += n
    assert float((got - want).abs().max()) < 1e-4
    # the last token's key is NaN: only its own slot may become NaN
    c.k[c.table[3, 39 // 16].long(), 39 % 16, 1] = math.nan
    got2 = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass)
    bad = torch.isnan(got2)
    assert bool(bad[3, 1, 39]) and int(bad.sum()) == 1
    assert torch.equal(got2[~bad], got[~bad])


def test_cache_mass_of_no_tokens_copies():
    c = Cache([5], 2, 64, 16, torch.float16, 8)
    mass = torch.rand(1, 2, 16, device=DEV)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device=DEV)
    lse = torch.zeros(0, 4, device=DEV)
    got = ops.cache_mass(q, lse, c.k, c.table, lengths_to_offsets([0]), c.lens, mass)
    assert torch.equal(got, mass)


# --------------------------------------------------------------------- edges of every call
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,new", [(64, [60, 50]), (128, [60, 50]), (128, [2, 3])])
def test_hidden_largest_values_do_not_count(dtype, d, new):
    """The type's largest number as a value that only the last token sees."""
    lens = [131, 80]
    c = Cache(lens, 2, d, 16, dtype, 8)
    for b, m in enumerate(lens):
        c.v[c.table[b, (m - 1) // 16].long(), (m - 1) % 16] = torch.finfo(dtype).max
    q = torch.randn(sum(new), 8, d, device=DEV, generator=_gen(5)).to(dtype)
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, return_lse=True)
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        s = slice(at, at + n - 1)  # all rows but the last, against keys without the last
        _check(out[s], lse[s], q[s], cache_rows(c.k, c.table, b, m)[:-1], cache_rows(c.v, c.table, b, m)[:-1], n - 1,
               m - 1, d**-0.5)
        at += n


@pytest.mark.parametrize("offsets", [[0, 40, 0, 40], [40, 40, 20, 0], [0, 1 << 30, -(1 << 30), 40]])
def test_offsets_that_do_not_rise_are_contained(offsets):
    """Results are nobody's, the status says so, and nothing outside the call is touched."""
    c = Cache([48, 64, 33], 2, 64, 16, torch.float16, 8)
    rows = torch.randn(60, 8, 64, device=DEV, generator=_gen(5)).half()
    q, k, v = rows[10:50], rows[10:50, :2], rows[10:50, 2:4]
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    big = torch.full((60, 8, 64), 7.0, dtype=torch.float16, device=DEV)
    mass = torch.ones(3, 2, c.table.shape[1] * 16, device=DEV)
    lse = torch.zeros(40, 8, device=DEV)
    kc, vc = c.k.clone(), c.v.clone()
    for call in (lambda s: ops.prompt_attention(q, k, v, off, out=big[10:50], status=s),
                 lambda s: ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, out=big[10:50], status=s),
                 lambda s: ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, out=big[10:50], max_new=1, status=s),
                 lambda s: ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass, status=s),
                 lambda s: ops.cache_append(k, v, kc, vc, c.table, off, c.lens, status=s)):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        call(status)
        assert int(status) == 0x402
    assert bool((big[:10] == 7).all()) and bool((big[50:] == 7).all())


def test_batches_of_padding_only():
    """Rows, but no sequence with tokens: outputs stay, masses are copied."""
    c = Cache([48, 64], 2, 64, 16, torch.float16, 8)
    q = torch.randn(70, 8, 64, device=DEV, generator=_gen(5)).half()
    k = q[:, :2]
    off, out = lengths_to_offsets([0, 0]), torch.full((70, 8, 64), 7.0, dtype=torch.float16, device=DEV)
    mass = torch.rand(2, 2, c.table.shape[1] * 16, device=DEV)
    before = c.k.clone()
    ops.prompt_attention(q, k, k, off, out=out)
    ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, out=out)
    ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, out=out, max_new=1)
    ops.cache_append(k, k, c.k, c.v, c.table, off, c.lens)
    assert bool((out == 7).all())
    assert torch.equal(c.k.view(torch.int16), before.view(torch.int16))
    assert torch.equal(ops.cache_mass(q, torch.zeros(70, 8, device=DEV), c.k, c.table, off, c.lens, mass), mass)


@pytest.mark.parametrize("new", [[1, 2, 1], [30, 1, 65]])
def test_padded_cache_batches_and_strided_outputs(new):
    lens = [90, 333, 70]
    c = Cache(lens, 2, 64, 16, torch.bfloat16, 8)
    t = sum(new)
    q = torch.randn(t + 9, 4, 64, device=DEV, generator=_gen(5)).bfloat16()
    q[t:] = math.nan
    big = torch.full((t + 9, 6, 80), 7.0, dtype=torch.bfloat16, device=DEV)
    off = lengths_to_offsets(new)
    ws = torch.empty(ops.serve_workspace_bytes(5, t + 100, 4, 2, 64), dtype=torch.uint8, device=DEV)
    out, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=max(new), out=big[:, 1:5, 8:72],
                                   return_lse=True, workspace=ws)
    _check_cache(out[:t], lse[:t], q, c, new, lens, 0.125)
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[:t, 1:5, 8:72] = False
    assert bool((big[keep] == 7).all())
    lse[t:] = math.nan
    mass = torch.rand(3, 2, c.table.shape[1] * 16, device=DEV)
    _check_mass(ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass), mass, q, lse, c, new, lens, 0.125)
    want = c.k.clone()
    kn = torch.randn(t + 9, 2, 64, device=DEV, generator=_gen(6)).bfloat16()
    kn[t:] = math.nan
    ops.cache_append(kn, kn, c.k, c.v, c.table, off, c.lens)
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        for i in range(n):
            j = m - n + i
            want[c.table[b, j // 16].long(), j % 16] = kn[at + i]
        at += n
    assert torch.equal(c.k.view(torch.int16), want.view(torch.int16))


def test_pages_shared_by_sequences():
    """A common prefix: two tables list the same pages, one lists a page twice."""
    c = Cache([96, 96, 96], 2, 64, 16, torch.float16, 8)
    c.table[1, :4] = c.table[0, :4]
    c.table[2, 3] = c.table[2, 1]
    lens = [96, 90, 96]
    c.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for new in ([1, 1, 1], [20, 40, 1]):
        q = torch.randn(sum(new), 4, 64, device=DEV, generator=_gen(5)).half()
        off = lengths_to_offsets(new)
        out, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=max(new), return_lse=True)
        _check_cache(out, lse, q, c, new, lens, 0.125)
        mass = torch.rand(3, 2, c.table.shape[1] * 16, device=DEV)
        _check_mass(ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass), mass, q, lse, c, new, lens, 0.125)


def test_the_most_sequences():
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 4, (1024,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 40, (1024,), generator=g))]
    new[1000], lens[1000] = 40, 70
    c = Cache(lens, 1, 32, 16, torch.float16, 8)
    q = torch.randn(sum(new), 2, 32, device=DEV, generator=_gen(5)).half()
    off = lengths_to_offsets(new)
    for hint in (1, 40):
        out, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=hint, return_lse=True)
        _check_cache(out, lse, q, c, new, lens, 32**-0.5)
    mass = torch.rand(1024, 1, c.table.shape[1] * 16, device=DEV)
    _check_mass(ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass), mass, q, lse, c, new, lens, 32**-0.5)
    pos = torch.arange(mass.shape[2], device=DEV, dtype=torch.int32).expand(mass.shape).contiguous()
    _check_evict(c, mass, pos, lens, 9, 2)
    out, lse = ops.prompt_attention(q, q[:, :1], q[:, 1:], off, return_lse=True)
    at = 0
    for n in new[:200] + [0]:
        s = slice(at, at + n)
        if n:
            _check(out[s], lse[s], q[s], q[s, :1], q[s, 1:], n, n, 32**-0.5)
        at += n


def test_calls_at_the_same_time():
    """Two streams, each with its own calls; results as alone."""
    def work(seed):
        c = Cache([700, 300, 1500], 2, 128, 32, torch.bfloat16, seed)
        new = [200, 1, 90]
        q = torch.randn(sum(new), 8, 128, device=DEV, generator=_gen(seed)).bfloat16()
        off = lengths_to_offsets(new)
        mass = torch.rand(3, 2, c.table.shape[1] * 32, device=DEV, generator=_gen(seed))
        pos = torch.arange(mass.shape[2], device=DEV, dtype=torch.int32).expand(mass.shape).contiguous()

        def run():
            out, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=200, return_lse=True)
            one = ops.cache_attention(q[:3], c.k, c.v, c.table, lengths_to_offsets([1, 1, 1]), c.lens, max_new=1)
            m = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass)
            own_k, own_v = c.k.clone(), c.v.clone()
            m2, p2, l2 = ops.cache_evict(m, pos, own_k, own_v, c.table, c.lens, 256, recent=16)
            pr = ops.prompt_attention(q, q[:, :2], q[:, 2:4], off)
            return out, lse, one, m, m2, p2, l2, pr, own_k.view(torch.int16), own_v.view(torch.int16)
        return run

    runs = [work(1), work(2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(runs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], g))


def test_captured_chunks_mass_and_eviction_follow_new_lengths():
    kv, heads, d, page, cap = 2, 8, 64, 16, 256
    c = Cache([cap] * 3, kv, d, page, torch.float16, 3)
    off = lengths_to_offsets([100, 20, 30])
    q = torch.zeros(150, heads, d, dtype=torch.float16, device=DEV)
    mass = torch.zeros(3, kv, cap, device=DEV)
    pos = torch.arange(cap, device=DEV, dtype=torch.int32).expand(3, kv, cap).contiguous()
    ws = torch.empty(ops.serve_workspace_bytes(3, 150, heads, kv, d), dtype=torch.uint8, device=DEV)

    def step():
        out, lse = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, return_lse=True, workspace=ws)
        prompt = ops.prompt_attention(q, q[:, :kv], q[:, kv:2 * kv], off, workspace=ws)
        m = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass)
        return out, lse, prompt, m, *ops.cache_evict(m, pos, c.k, c.v, c.table, c.lens, 64, recent=8)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, (new, lens) in enumerate([([100, 20, 30], [100, 256, 31]), ([1, 0, 140], [1, 77, 200]), ([5, 3, 2], [5, 3, 256])]):
        g = _gen(20 + i)
        q.copy_(torch.randn(q.shape, device=DEV, generator=g))
        mass.copy_(torch.rand(mass.shape, device=DEV, generator=g))
        c.lens.copy_(torch.tensor(lens))
        off.copy_(lengths_to_offsets(new))
        c.k.copy_(torch.randn(c.k.shape, device=DEV, generator=g))
        c.v.copy_(torch.randn(c.v.shape, device=DEV, generator=g))
        k0, v0 = c.k.clone(), c.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed, k1, v1 = [x.clone() for x in got], c.k.clone(), c.v.clone()
        c.k.copy_(k0), c.v.copy_(v0)
        t = sum(new)
        _check_cache(replayed[0][:t], replayed[1][:t], q, c, new, lens, 0.125)
        _check_mass(replayed[3], mass, q, replayed[1], c, new, lens, 0.125)
        for j, (a, b) in enumerate(zip(replayed, step())):
            assert torch.equal(a[:t], b[:t]) if j < 3 else torch.equal(a, b)
        assert torch.equal(k1, c.k) and torch.equal(v1, c.v)


def test_requires_grad_and_wide_integers():
    c = Cache([20, 30], 2, 64, 16, torch.float16, 8)
    q = torch.randn(2, 4, 64, device=DEV, generator=_gen(5)).half()
    off = lengths_to_offsets([1, 1])
    for name in ("q", "k", "v", "out"):
        args = dict(q=q, k=q[:, :2], v=q[:, 2:], out=torch.empty_like(q))
        args[name] = args[name].clone().requires_grad_()
        with pytest.raises(ValueError, match="inference only"):
            ops.prompt_attention(args["q"], args["k"], args["v"], off, out=args["out"])
        with torch.no_grad():
            ops.prompt_attention(args["q"], args["k"], args["v"], off, out=args["out"])
    with pytest.raises(ValueError, match="inference only"):
        ops.cache_attention(q, c.k, c.v.clone().requires_grad_(), c.table, off, c.lens)
    mass = torch.rand(2, 2, c.table.shape[1] * 16, device=DEV)
    with pytest.raises(ValueError, match="inference only"):
        ops.cache_mass(q, torch.zeros(2, 4, device=DEV), c.k, c.table, off, c.lens, mass.clone().requires_grad_())
    pos = torch.arange(mass.shape[2], device=DEV, dtype=torch.int32).expand(mass.shape).contiguous()
    for keep, recent in ((2**32 + 1, 0), (2**31, 2**31)):
        _check_evict(c, mass, pos, [20, 30], keep, recent)
    for keep, recent in ((0, 0), (-(2**32) + 3, 0), (4, 5), (2**33, 2**34), (4, -1)):
        with pytest.raises(ValueError, match="keep"):
            ops.cache_evict(mass, pos, c.k, c.v, c.table, c.lens, keep, recent=recent)
    want = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens)
    assert torch.equal(want, ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=2**40))
    with pytest.raises(ValueError, match="max_new"):
        ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=-1)
    with pytest.raises(ValueError, match="1-D"):
        ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, workspace=torch.empty(2, 1 << 24, dtype=torch.uint8, device=DEV))


# ---------------------------------------------------------------------------- all together
@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_steps_with_a_budget(dtype):
    """A user's loop: attend to the prompts, cache them, gather their mass, cut the cache to
    a budget, then single tokens -- append, attend, gather, evict -- against a plain model of
    the same cache that holds 64-bit masses and Python lists of kept tokens."""
    heads, kv, d, page, keep, recent = 6, 2, 64, 16, 48, 8
    lens = [100, 30, 61]
    b, g, scale = len(lens), 3, 64**-0.5
    gen = _gen(77)
    per = 8
    kc = torch.zeros(b * per, page, kv, d, dtype=dtype, device=DEV)
    vc = torch.zeros_like(kc)
    table = torch.randperm(b * per, device=DEV, generator=gen).to(torch.int32).view(b, per)
    cap = per * page
    mass, pos = torch.zeros(b, kv, cap, device=DEV), torch.full((b, kv, cap), -1, dtype=torch.int32, device=DEV)
    seen = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cache_lens = seen.clone()
    rand = lambda t, h: torch.randn(t, h, d, device=DEV, generator=gen).to(dtype)  # noqa: E731
    # model: per (sequence, head) the keys and values that are kept, by position
    model = [[{} for _ in range(kv)] for _ in range(b)]

    def attend_model(q, i, hh):
        h = hh // g
        items = model[i][h]
        k = torch.stack([items[p][0] for p in sorted(items)]).double()
        v = torch.stack([items[p][1] for p in sorted(items)]).double()
        w = torch.softmax(k @ q.double() * scale, 0)
        return w @ v, dict(zip(sorted(items), w.tolist()))

    t = sum(lens)
    q, k, v = rand(t, heads), rand(t, kv), rand(t, kv)
    off = lengths_to_offsets(lens)
    out, lse = ops.prompt_attention(q, k, v, off, return_lse=True)
    ops.cache_append(k, v, kc, vc, table, off, cache_lens, positions=pos, mass=mass, seen=seen)
    chunk, chunk_lse = ops.cache_attention(q, kc, vc, table, off, cache_lens, max_new=max(lens), return_lse=True)
    u = torch.finfo(dtype).eps
    assert float((chunk.double() - out.double()).abs().max()) <= 4 * u * float(v.abs().max())
    assert float((chunk_lse - lse).abs().max()) < 1e-4
    mass = ops.cache_mass(q, lse, kc, table, off, cache_lens, mass, out=mass)
    at = 0
    for i, n in enumerate(lens):
        for h in range(kv):
            for p in range(n):
                model[i][h][p] = (k[at + p, h], v[at + p, h])
        at += n
    assert float((mass.sum(2).cpu() - torch.tensor([[n * g] * kv for n in lens], dtype=torch.float32)).abs().max()) < 0.01
    step_off = lengths_to_offsets([1] * b)
    for step in range(12):
        # cut to the budget; the model follows the choice that the operator reports
        old_pos, old_mass, old_lens = pos.clone(), mass.clone(), cache_lens.tolist()
        mass, pos, cache_lens = ops.cache_evict(mass, pos, kc, vc, table, cache_lens, keep, recent=recent)
        for i in range(b):
            for h in range(kv):
                hole, mover = evict_choice(old_mass[i, h], old_pos[i, h], old_lens[i], keep, recent)
                gone = {int(old_pos[i, h, j]) for j in hole}
                gone |= {int(old_pos[i, h, j]) for j in range(keep, old_lens[i])} - {int(old_pos[i, h, j]) for j in mover}
                for p in gone:
                    del model[i][h][p]
                n = int(cache_lens[i])
                assert sorted(pos[i, h, :n].tolist()) == sorted(model[i][h])
        q, k, v = rand(b, heads), rand(b, kv), rand(b, kv)
        seen += 1
        cache_lens = cache_lens + 1
        ops.cache_append(k, v, kc, vc, table, step_off, cache_lens, positions=pos, mass=mass, seen=seen)
        out, lse = ops.cache_attention(q, kc, vc, table, step_off, cache_lens, max_new=1, return_lse=True)
        before = mass.clone()
        ops.cache_mass(q, lse, kc, table, step_off, cache_lens, mass, max_new=1, out=mass)
        for i in range(b):
            for h in range(kv):
                model[i][h][int(seen[i]) - 1] = (k[i, h], v[i, h])
            gained = {}
            for hh in range(heads):
                ref, w = attend_model(q[i, hh], i, hh)
                assert float((out[i, hh].double() - ref).abs().max()) <= 2 * u * float(vc.abs().max())
                for p, x in w.items():
                    gained[(hh // g, p)] = gained.get((hh // g, p), 0) + x
            for h in range(kv):
                for j in range(int(cache_lens[i])):
                    p = int(pos[i, h, j])
                    assert abs(float(mass[i, h, j] - before[i, h, j]) - gained[(h, p)]) < 1e-4
