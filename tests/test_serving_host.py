"""CPU: what the serving operators refuse, through the C entry points (nothing is launched)
and through the Python wrappers."""
import ctypes

import pytest
import torch

from tttj_2026_b200 import _lib, ops

A = 1 << 20  # any aligned address: refusals look at it, never through it


def _seqs(**kw):
    base = dict(seq_offsets=A, cache_lens=A, page_table=A, table_stride=8, batch=2, tokens=5, pages_per_seq=8,
                page_size=16, num_pages=16, dtype=_lib.DTYPE_F16, heads=8, kv_heads=2, head_dim=64, status=None)
    base.update(kw)
    return _lib.TttjSeqs(*[base[n] for n, _ in _lib.TttjSeqs._fields_])


def _rows(data=A, tok=512, head=64):
    return ctypes.byref(_lib.TttjRows(data, tok, head))


def _pages(data=A, page=2048, slot=128, head=64):
    return ctypes.byref(_lib.TttjPages(data, page, slot, head))


def _attend(s, q=None, kc=None, out=None, scale=0.125, ws=A, nbytes=1 << 30, max_new=1):
    return _lib.lib().tttj_cache_attention(ctypes.byref(s), q or _rows(), kc or _pages(), _pages(), out or _rows(),
                                           None, max_new, scale, ws, nbytes, None)


def _refused(rc, text):
    assert rc == _lib.TTTJ_ERR_INVALID
    assert text in _lib.lib().tttj_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=_lib.DTYPE_F32), "fp16 or bf16"), (dict(head_dim=48), "head_dim=48"), (dict(heads=9), "heads=9"),
    (dict(heads=130, kv_heads=2), "group"), (dict(kv_heads=0), "heads"), (dict(batch=0), "batch"),
    (dict(batch=1025), "batch"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 29), "tokens"),
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(pages_per_seq=0), "pages_per_seq"), (dict(pages_per_seq=1 << 28), "pages_per_seq"),
    (dict(num_pages=0), "num_pages"), (dict(table_stride=7), "overlap"), (dict(seq_offsets=None), "seq_offsets"),
    (dict(cache_lens=None), "cache_lens"), (dict(page_table=None), "page_table"),
])
def test_sequences_refused(kw, text):
    _refused(_attend(_seqs(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=_rows(tok=0)), "q strides"), (dict(q=_rows(tok=516)), "q strides"), (dict(q=_rows(head=-64)), "q strides"),
    (dict(q=_rows(data=A + 8)), "q must be 16-byte"), (dict(q=_rows(data=None)), "null q"),
    (dict(out=_rows(head=0)), "out strides"), (dict(kc=_pages(slot=0)), "k_cache strides"),
    (dict(kc=_pages(page=-8)), "k_cache strides"), (dict(kc=_pages(data=A + 2)), "k_cache must be 16-byte"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(ws=None), "workspace"), (dict(nbytes=16), "workspace too small"),
    (dict(ws=A + 16), "256-byte"), (dict(max_new=-1), "max_new"),
])
def test_attention_arguments_refused(kw, text):
    _refused(_attend(_seqs(), **kw), text)


def test_no_tokens_is_nothing_to_do():
    s = _seqs(tokens=0)
    assert _attend(s, q=_rows(data=None), out=_rows(data=None)) == 0
    assert _lib.lib().tttj_cache_append(ctypes.byref(s), _rows(data=None), _rows(data=None), _pages(), _pages(),
                                        None, None, None, None) == 0


def _evict(s, keep=8, recent=0, mass=A, mass_out=2 * A, ws=A, nbytes=1 << 30):
    return _lib.lib().tttj_cache_evict(ctypes.byref(s), _pages(), _pages(), mass, A, keep, recent, mass_out, 2 * A,
                                       2 * A, ws, nbytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(keep=0), "keep"), (dict(recent=-1), "recent"), (dict(recent=9), "recent"), (dict(mass=None), "null"),
    (dict(mass_out=A), "outputs may not"), (dict(nbytes=8), "workspace too small"), (dict(ws=A + 8), "256-byte"),
])
def test_evict_arguments_refused(kw, text):
    _refused(_evict(_seqs(), **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=_rows(tok=0)), "q strides"), (dict(q=_rows(data=A + 8)), "q must be 16-byte"), (dict(lse=None), "null"),
    (dict(kc=_pages(slot=0)), "k_cache strides"), (dict(mass=None), "null"), (dict(out=None), "null"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(max_new=-1), "max_new"),
    (dict(s=_seqs(batch=1025)), "batch"), (dict(s=_seqs(cache_lens=None)), "cache_lens"),
])
def test_mass_arguments_refused(kw, text):
    a = dict(s=_seqs(), q=_rows(), lse=A, kc=_pages(), mass=A, out=A, max_new=0, scale=0.125) | kw
    _refused(_lib.lib().tttj_cache_mass(ctypes.byref(a["s"]), a["q"], a["lse"], a["kc"], a["mass"], a["out"],
                                        a["max_new"], a["scale"], None), text)


def test_packed_arguments_have_the_c_layout():
    seqs = [A, 2 * A, 3 * A, 1 << 40, *range(1, 10), 4 * A]
    assert ops._pack_seqs(*seqs) == bytes(_lib.TttjSeqs(*seqs))
    assert ops._pack_rows(A, 1 << 40, -3) == bytes(_lib.TttjRows(A, 1 << 40, -3))
    assert ops._pack_pages(A, 1 << 40, 5, 6) == bytes(_lib.TttjPages(A, 1 << 40, 5, 6))


def test_workspace_sizes():
    L = _lib.lib()
    assert L.tttj_serve_workspace_bytes(ctypes.byref(_seqs())) > 0
    assert L.tttj_serve_workspace_bytes(ctypes.byref(_seqs(head_dim=40))) == 0
    s = _seqs()
    # moves: at most min(keep, slots - keep) of 8 bytes per head
    assert L.tttj_cache_evict_workspace_bytes(ctypes.byref(s), 100) >= 4 * 28 * 8
    assert L.tttj_cache_evict_workspace_bytes(ctypes.byref(s), 10**6) > 0
    assert ops.serve_workspace_bytes(2, 5, 8, 2, 64) == L.tttj_serve_workspace_bytes(ctypes.byref(s))
    with pytest.raises(ValueError, match="head_dim=40"):
        ops.serve_workspace_bytes(2, 5, 8, 2, 40)
    assert L.tttj_cache_evict_workspace_bytes(ctypes.byref(s), 0) == 0


def test_wrappers_refuse_before_any_launch():
    q = torch.zeros(4, 8, 64, dtype=torch.float16)
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.prompt_attention(q, k, k, off)
    with pytest.raises(ValueError, match="float16, bfloat16"):
        ops.prompt_attention(q.float(), k.float(), k.float(), off)
    with pytest.raises(ValueError, match="tokens, heads, head_dim"):
        ops.prompt_attention(q[0], k, k, off)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="k_cache"):
        ops.cache_attention(q, cache[0], cache, off, off, off)
    with pytest.raises(ValueError, match="k_cache"):
        ops.cache_append(k, k, cache[0], cache, off, off, off)
    with pytest.raises(ValueError, match="k_cache"):
        ops.cache_evict(cache, cache, cache[0], cache, off, off, 4)
    with pytest.raises(ValueError, match="k_cache"):
        ops.cache_mass(q, q, cache[0], off, off, off, q)
