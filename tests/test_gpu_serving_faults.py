"""GPU: serving operators, calls that went wrong once: tokens behind the table, tensors with
gradients or tangents, weights outside fp32's range, calls of two threads, device waits that
give up, a captured step that carries its own state.  Tolerances as in test_gpu_serving.py."""
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from serving_reference import attention_rows, cache_rows, lengths_to_offsets
from test_gpu_serving import Cache, _check, _gen
from tttj_2026_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# -------------------------------------------------------------------------------- append
@pytest.mark.parametrize("with_seen", [False, True])
@pytest.mark.parametrize("length", [65, 66, 67, 1 << 30, 2**31 - 1])
def test_append_keeps_live_slots_when_a_length_exceeds_the_table(length, with_seen):
    """64 slots, three new tokens: those whose slot is not in the table are dropped, and no slot in
    front of the new tokens changes."""
    new, lens = [3, 1], [length, 64]
    c = Cache([64, 64], 2, 64, 16, torch.float16, 3)
    c.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want_k, want_v = c.k.clone(), c.v.clone()
    k = torch.randn(4, 2, 64, device=DEV, generator=_gen(1)).half()
    pos = torch.full((2, 2, 64), 77, dtype=torch.int32, device=DEV)
    mass = torch.full((2, 2, 64), 5.0, device=DEV)
    want_pos, want_mass = pos.clone(), mass.clone()
    seen = torch.tensor([1000, 2000], dtype=torch.int32, device=DEV) if with_seen else None
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        for i in range(n):
            slot = m - n + i
            if slot < 64:
                page = c.table[b, slot // 16].long()
                want_k[page, slot % 16], want_v[page, slot % 16] = k[at + i], k[at + i] + 1
                want_pos[b, :, slot] = (1000 * (b + 1) if with_seen else m) - n + i
                want_mass[b, :, slot] = 0
        at += n
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.cache_append(k, k + 1, c.k, c.v, c.table, lengths_to_offsets(new), c.lens, positions=pos, mass=mass, seen=seen,
                     status=status)
    assert int(status) == 0x402
    assert torch.equal(c.k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), want_v.view(torch.int16))
    assert torch.equal(pos, want_pos) and torch.equal(mass, want_mass)


def test_append_says_that_it_dropped_tokens_before_the_first_slot():
    c = Cache([64, 64], 2, 64, 16, torch.float16, 3)
    k = torch.randn(6, 2, 64, device=DEV, generator=_gen(1)).half()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for lens, want in (([4, 2], 0), ([3, 2], 0x402), ([4, 0], 0x402), ([4, -1], 0x402)):
        status.zero_()
        c.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        ops.cache_append(k, k, c.k, c.v, c.table, lengths_to_offsets([4, 2]), c.lens, status=status)
        assert int(status) == want, lens


# ----------------------------------------------------------------------------- gradients
def _call_all(q, k, lse, c, mass):
    """Every operator, as a list of (name, call of its floating-point tensors, those tensors)."""
    off = lengths_to_offsets([1, 1])
    pos = torch.arange(mass.shape[2], device=DEV, dtype=torch.int32).expand(mass.shape).contiguous()
    return [
        ("prompt", lambda a: ops.prompt_attention(a[0], a[1], a[2], off, out=a[3]), [q, k, k, torch.empty_like(q)]),
        ("attend", lambda a: ops.cache_attention(a[0], a[1], a[2], c.table, off, c.lens, out=a[3]),
         [q, c.k, c.v, torch.empty_like(q)]),
        ("append", lambda a: ops.cache_append(a[0], a[1], a[2], a[3], c.table, off, c.lens, mass=a[4]),
         [k, k, c.k.clone(), c.v.clone(), mass.clone()]),
        ("mass", lambda a: ops.cache_mass(a[0], a[1], a[2], c.table, off, c.lens, a[3], out=a[4]),
         [q, lse, c.k, mass, mass.clone()]),
        ("evict", lambda a: ops.cache_evict(a[0], pos, a[1], a[2], c.table, c.lens, 16),
         [mass, c.k.clone(), c.v.clone()]),
    ]


def _grad_inputs():
    c = Cache([20, 30], 2, 64, 16, torch.float16, 8)
    q = torch.randn(2, 4, 64, device=DEV, generator=_gen(5)).half()
    lse = torch.zeros(2, 4, device=DEV)
    mass = torch.rand(2, 2, c.table.shape[1] * 16, device=DEV)
    return q, q[:, :2], lse, c, mass


def test_every_tensor_with_a_gradient_is_refused():
    for name, call, tensors in _call_all(*_grad_inputs()):
        call(tensors)
        for i in range(len(tensors)):
            a = [t.clone() for t in tensors]
            a[i].requires_grad_()
            with pytest.raises(ValueError, match="inference only"):
                call(a)
            with torch.no_grad():
                call(a)


def test_every_tensor_with_a_tangent_is_refused():
    """Forward-mode derivatives would be dropped silently."""
    fwd = torch.autograd.forward_ad
    for name, call, tensors in _call_all(*_grad_inputs()):
        for i in range(len(tensors)):
            with fwd.dual_level():
                a = list(tensors)
                a[i] = fwd.make_dual(tensors[i].clone(), torch.ones_like(tensors[i]))
                with pytest.raises(ValueError, match="inference only"):
                    call(a)
                call(tensors)  # no tangent: served
        call(tensors)


# ---------------------------------------------------------------------------------- mass
@pytest.mark.parametrize("shift", [0.0, 5.0, 40.0, 86.0, 88.0, 95.0, 400.0, -60.0, -300.0])
def test_mass_far_from_the_log_sum_exp(shift):
    """One row after the other (each column of the accumulator) has an lse that lies `shift` below its
    largest score, the others' weights are zero: weights grow up to fp32's overflow, and to
    infinity beyond; weights of zero leave a mass of zero."""
    d, n, m, heads = 64, 3, 900, 16
    c = Cache([m], 2, d, 16, torch.float16, 8)
    q = torch.randn(n, heads, d, device=DEV, generator=_gen(5)).half()
    off = lengths_to_offsets([n])
    k = cache_rows(c.k, c.table, 0, m).double()
    s = torch.einsum("nhd,mhd->nhm", q.double(), k.repeat_interleave(heads // 2, 1)) * d**-0.5
    hidden = torch.ones(n, m, dtype=torch.bool, device=DEV).triu(m - n + 1)
    s.masked_fill_(hidden[:, None], -math.inf)
    sa = torch.einsum("nhd,mhd->nhm", q.double().abs(), k.abs().repeat_interleave(heads // 2, 1)) * d**-0.5
    zeros = torch.zeros(1, 2, c.table.shape[1] * 16, device=DEV)
    big = torch.finfo(torch.float32).max
    for i in range(n):
        for h in range(heads):
            lse = torch.full((n, heads), 1e4, device=DEV)
            lse[i, h] = s[i, h].max() - shift
            got = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, zeros)[0, :, :m].double()
            assert bool((got[1 - h // 8] == 0).all())
            got, g = got[h // 8], lse[i, h].double()
            want = torch.exp(s[i, h] - g)
            # its score's error (an fp32 sum of d products), the exponent's roundings, and what is
            # too small for a normal number
            rel = d * 2.0**-24 * sa[i, h] + 2.0**-21 * (1 + torch.nan_to_num(s[i, h].abs(), posinf=0) + g.abs())
            tol = want * rel + 2.0**-125
            assert not bool(torch.isnan(got).any())
            assert bool(torch.isposinf(got)[want - tol > big].all())
            fits = want + tol < big
            err = (got - want).abs()
            assert bool((err <= tol)[fits].all()), f"{float((err / tol)[fits].max()):.2f} times the tolerance"
            if shift == -300.0:
                assert bool((got == 0).all())


# ------------------------------------------------------------------------------- threads
@pytest.mark.parametrize("op", ["attend", "mass"])
def test_two_threads_with_batches_of_different_sizes(op, monkeypatch):
    """Calls need shared memory by their number of sequences: neither thread's launch may depend on
    the other's."""
    recorded = []
    real = ops._call

    def record(device, fn, *args):
        recorded.append((fn, args))
        return real(device, fn, *args)

    monkeypatch.setattr(ops, "_call", record)
    kept = []
    for batch in (1, 1024):
        c = Cache([17] * batch, 1, 64, 32, torch.float16, batch)
        q = torch.randn(batch, 2, 64, device=DEV, generator=_gen(5)).half()
        off = lengths_to_offsets([1] * batch)
        mass, lse = torch.zeros(batch, 1, c.table.shape[1] * 32, device=DEV), torch.zeros(batch, 2, device=DEV)
        ws = torch.empty(ops.serve_workspace_bytes(batch, batch, 2, 1, 64), dtype=torch.uint8, device=DEV)
        if op == "mass":
            out = ops.cache_mass(q, lse, c.k, c.table, off, c.lens, mass, max_new=1)
        else:
            out = ops.cache_attention(q, c.k, c.v, c.table, off, c.lens, max_new=1, workspace=ws)
        kept.append((c, q, off, mass, lse, ws, out))
    torch.cuda.synchronize()
    failed = [0, 0]

    def loop(i):
        torch.cuda.set_device(0)
        fn, args = recorded[i]
        stream = torch.cuda.Stream()
        for _ in range(300):
            for _ in range(100):
                failed[i] += fn(*args, stream.cuda_stream) != 0
            stream.synchronize()

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failed == [0, 0]


# --------------------------------------------------------------------- failure detection
@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("with_status", [False, True])
def test_a_wait_that_gave_up_is_reported_by_the_next_call(which, with_status):
    """A 2 ms wait on nothing, reported as a kernel's would be: the next call raises once and launches
    nothing, the one after it is served."""
    name, call, tensors = _call_all(*_grad_inputs())[which]
    want = call(tensors)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.serve_selftest_timeout(torch.device(DEV), status=status if with_status else None)
    torch.cuda.synchronize()
    assert int(status) == (0x403 if with_status else 0)
    before = [t.clone() for t in tensors]
    with pytest.raises(RuntimeError, match="timed out"):
        call(tensors)
    torch.cuda.synchronize()
    for a, b in zip(before, tensors):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
    got = call(tensors)
    if name in ("prompt", "attend"):
        assert torch.equal(got, want)


def test_serve_status_raises_once():
    assert ops.serve_status(torch.device(DEV)) == 0
    ops.serve_selftest_timeout(torch.device(DEV))
    with pytest.raises(RuntimeError, match="timed out"):
        ops.serve_status(torch.device(DEV))
    assert ops.serve_status(torch.device(DEV)) == 0
    with pytest.raises(ValueError, match="1 s"):
        ops.serve_selftest_timeout(torch.device(DEV), limit_ns=10**10)


def test_first_call_of_a_process_under_capture():
    """The device's word is made by the first call, which may be a captured one."""
    code = """
import torch, optimized_transformer
from tttj_2026_b200 import ops
g = torch.Generator(device="cuda").manual_seed(1)
kc = torch.randn(8, 16, 2, 64, device="cuda", generator=g).half()
q = torch.randn(2, 4, 64, device="cuda", generator=g).half()
table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
off = torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)
lens = torch.tensor([30, 64], device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.cache_attention(q, kc, kc, table, off, lens, max_new=1)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, ops.cache_attention(q, kc, kc, table, off, lens, max_new=1))
print("served")
"""
    root = Path(__file__).resolve().parent.parent
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "served" in res.stdout, res.stderr[-2000:]


# --------------------------------------------------------------------- a captured step
def test_a_captured_step_carries_its_state():
    """Evict, append, attend, gather in one graph, as INTEGRATION.md shows it: eviction makes new
    tensors, so the step ends by copying them into those that the next replay reads.  Replays follow
    the same steps run one by one on tensors of their own, bit for bit."""
    heads, kv, d, page, per, keep, recent = 8, 2, 64, 16, 6, 40, 6
    lens0 = [90, 12, 41]
    b, cap = len(lens0), per * page
    gen = _gen(7)
    kc = torch.randn(b * per, page, kv, d, device=DEV, generator=gen).half()
    vc = torch.randn(b * per, page, kv, d, device=DEV, generator=gen).half()
    table = torch.randperm(b * per, device=DEV, generator=gen).to(torch.int32).view(b, per)
    lens = torch.tensor(lens0, dtype=torch.int32, device=DEV)
    live = torch.arange(cap, device=DEV)[None, None] < lens[:, None, None]
    mass = torch.where(live, torch.rand(b, kv, cap, device=DEV, generator=gen), 0.0)
    pos = torch.where(live, torch.arange(cap, device=DEV)[None, None].expand(b, kv, cap), -1).to(torch.int32).contiguous()
    seen, off = lens.clone(), lengths_to_offsets([1] * b)
    q = torch.zeros(b, heads, d, dtype=torch.float16, device=DEV)
    k, v = torch.zeros(b, kv, d, dtype=torch.float16, device=DEV), torch.zeros(b, kv, d, dtype=torch.float16, device=DEV)

    def step():
        m, p, n = ops.cache_evict(mass, pos, kc, vc, table, lens, keep, recent=recent)
        mass.copy_(m), pos.copy_(p), lens.copy_(n + 1), seen.add_(1)
        ops.cache_append(k, v, kc, vc, table, off, lens, positions=pos, mass=mass, seen=seen)
        out, lse = ops.cache_attention(q, kc, vc, table, off, lens, max_new=1, return_lse=True)
        ops.cache_mass(q, lse, kc, table, off, lens, mass, max_new=1, out=mass)
        return out, lse

    state = (mass, pos, lens, seen, kc, vc)
    start = [x.clone() for x in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_lse = step()
    for x, y in zip(state, start):
        x.copy_(y)
    m, p, n, s, k2, v2 = [x.clone() for x in start]
    for i in range(60):  # past the budget, and every sequence evicts
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV, generator=gen))
        graph.replay()
        m, p, n = ops.cache_evict(m, p, k2, v2, table, n, keep, recent=recent)
        n, s = n + 1, s + 1
        ops.cache_append(k, v, k2, v2, table, off, n, positions=p, mass=m, seen=s)
        out, lse = ops.cache_attention(q, k2, v2, table, off, n, max_new=1, return_lse=True)
        ops.cache_mass(q, lse, k2, table, off, n, m, max_new=1, out=m)
        assert torch.equal(got, out) and torch.equal(got_lse, lse), i
        for x, y in zip(state, (m, p, n, s, k2, v2)):
            assert torch.equal(x, y), i
    assert n.tolist() == [keep + 1] * b
    assert s.tolist() == [x + 60 for x in lens0]
    assert ops.serve_status(torch.device(DEV)) == 0


# ---------------------------------------------------------------- log-sum-exps, many prompts
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_log_sum_exp_of_rows_that_see_a_nan(d):
    """NaN for a row whose scores hold one, on every path, split keys among them; a number elsewhere."""
    def check(lse, q, k, n, m):
        _, want = attention_rows(q, k, torch.zeros_like(k), n, m, d**-0.5)
        assert torch.equal(torch.isnan(lse), torch.isnan(want))
        assert torch.equal(torch.isneginf(lse.double()), torch.isneginf(want))
        assert 0 < int(torch.isnan(want).sum()) < want.numel()

    q = torch.randn(200, 4, d, device=DEV, generator=_gen(5)).half()
    k = torch.randn(200, 2, d, device=DEV, generator=_gen(6)).half()
    for at in (3, 130, 199):
        bad = k.clone()
        bad[at, 1, 0] = math.nan
        _, lse = ops.prompt_attention(q, bad, k, lengths_to_offsets([200]), return_lse=True)
        check(lse, q, bad, 200, 200)
    for m in (300, 9001):
        for n in (3, 150):
            for back in (0, 1, 100):
                c = Cache([m], 2, d, 16, torch.float16, 8)
                slot = m - n if back == 100 else m - 1 - back
                c.k[c.table[0, slot // 16].long(), slot % 16, 1, 2] = math.nan
                qn = q[:n]
                _, lse = ops.cache_attention(qn, c.k, c.v, c.table, lengths_to_offsets([n]), c.lens, return_lse=True)
                check(lse, qn, cache_rows(c.k, c.table, 0, m), n, m)


def test_every_prompt_of_the_most_sequences():
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 4, (1024,), generator=g).tolist()
    new[1000], new[1023], new[600] = 40, 130, 0
    q = torch.randn(sum(new), 4, 32, device=DEV, generator=_gen(5)).half()
    out, lse = ops.prompt_attention(q[:, :2], q[:, 2:3], q[:, 3:], lengths_to_offsets(new), return_lse=True)
    at = 0
    for n in new:
        s = slice(at, at + n)
        if n:
            _check(out[s], lse[s], q[s, :2], q[s, 2:3], q[s, 3:], n, n, 32**-0.5)
        at += n
