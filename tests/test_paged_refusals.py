"""What the paged-cache and draft-verification entry points refuse.  The C checks come before any CUDA
call, so they run without a GPU: the pointers below are never followed."""
from __future__ import annotations

import ctypes as C
import math

import pytest

P = 1 << 20  # an address with every alignment


def append_args(pkg, **ch):
    cache = dict(k=P, v=P, k_scale=P, v_scale=P, num_pages=8, page_size=64, kv_heads=8)
    batch = dict(cu_q=P, seq_len=P, page_table=P, num_seqs=2, table_stride=4, total_q=3, max_q=2, max_len=200)
    args = dict(q=P, k_new=P, v_new=P, q_stride=48 * 128, k_stride=1024, v_stride=1024, in_type=0, heads=48, cos=P, sin=P,
                rope_dim=64, positions=200, q_out=P, out_type=1)
    for name, value in ch.items():
        where = cache if name in cache and name not in ("q",) else batch if name in batch else args
        assert name in where, name
        where[name] = value
    c = pkg.MmrsPagedCache(*cache.values())
    b = pkg.MmrsPagedBatch(*batch.values())
    return (C.byref(c), C.byref(b), *args.values(), None), (c, b)


@pytest.mark.parametrize("ch,name", [
    (dict(k=None), "ARG"), (dict(v=None), "ARG"), (dict(k_scale=None), "ARG"), (dict(k=P + 64), "ARG"),
    (dict(page_size=48), "UNSUPPORTED"), (dict(page_size=256), "UNSUPPORTED"), (dict(num_pages=0), "ARG"),
    (dict(kv_heads=0), "ARG"), (dict(num_pages=1 << 24), "UNSUPPORTED"), (dict(num_seqs=-1), "ARG"),
    (dict(num_seqs=1025), "UNSUPPORTED"), (dict(cu_q=None), "ARG"), (dict(seq_len=None), "ARG"),
    (dict(page_table=None), "ARG"), (dict(max_q=0), "ARG"), (dict(max_len=0), "ARG"), (dict(table_stride=3), "ARG"),
    (dict(total_q=-1), "ARG"), (dict(in_type=3), "UNSUPPORTED"), (dict(in_type=-1), "UNSUPPORTED"),
    (dict(out_type=0), "UNSUPPORTED"), (dict(rope_dim=130), "UNSUPPORTED"), (dict(rope_dim=7), "UNSUPPORTED"),
    (dict(q_out=None), "ARG"), (dict(q=None), "ARG"), (dict(k_new=None), "ARG"), (dict(v_new=None), "ARG"),
    (dict(cos=None), "ARG"), (dict(positions=199), "ARG"), (dict(k_stride=1023), "ARG"), (dict(k_stride=512), "ARG"),
    (dict(v_stride=1026), "ARG"), (dict(q_stride=47 * 128), "ARG"), (dict(q_stride=48 * 128 + 4, in_type=1), "ARG"),
    (dict(k_new=P + 8), "ARG"), (dict(q_out=P + 8), "ARG"), (dict(heads=0), "ARG"),
])
def test_append(pkg, ch, name):
    args, _keep = append_args(pkg, **ch)
    assert pkg.lib().mmrs_paged_append(*args) == getattr(pkg, "MMRS_ERR_" + name)


def test_append_of_nothing(pkg):
    for ch in (dict(num_seqs=0, cu_q=None, seq_len=None, page_table=None), dict(total_q=0, k_new=None, v_new=None)):
        args, _keep = append_args(pkg, **ch)
        assert pkg.lib().mmrs_paged_append(*args) == pkg.MMRS_OK


def attend_args(pkg, **ch):
    cache = dict(k=P, v=P, k_scale=P, v_scale=P, num_pages=8, page_size=64, kv_heads=8)
    batch = dict(cu_q=P, seq_len=P, page_table=P, num_seqs=2, table_stride=4, total_q=3, max_q=2, max_len=200)
    args = dict(q=P, q_stride=48 * 128, type=1, heads=48, scale=0.1, window=0, sinks=0, out=P, lse=None, ws=P, ws_bytes=1 << 40)
    for name, value in ch.items():
        where = next(d for d in (cache, batch, args) if name in d)
        where[name] = value
    c = pkg.MmrsPagedCache(*cache.values())
    b = pkg.MmrsPagedBatch(*batch.values())
    return (C.byref(c), C.byref(b), *args.values(), None), (c, b)


@pytest.mark.parametrize("ch,name", [
    (dict(k=None), "ARG"), (dict(page_size=8), "UNSUPPORTED"), (dict(type=0), "UNSUPPORTED"), (dict(type=3), "UNSUPPORTED"),
    (dict(heads=47), "UNSUPPORTED"), (dict(heads=0), "UNSUPPORTED"), (dict(heads=17 * 8), "UNSUPPORTED"),
    (dict(scale=math.nan), "ARG"), (dict(scale=math.inf), "ARG"), (dict(window=-1), "ARG"), (dict(sinks=-1), "ARG"),
    (dict(q=None), "ARG"), (dict(out=None), "ARG"), (dict(q=P + 8), "ARG"), (dict(out=P + 4), "ARG"),
    (dict(q_stride=48 * 128 + 4), "ARG"), (dict(q_stride=47 * 128), "ARG"), (dict(ws=None), "ARG"),
    (dict(ws=P + 128), "ARG"), (dict(ws_bytes=255), "ARG"),
])
def test_attend(pkg, ch, name):
    args, _keep = attend_args(pkg, **ch)
    assert pkg.lib().mmrs_paged_attend(*args) == getattr(pkg, "MMRS_ERR_" + name)


def test_attend_workspace(pkg):
    need = pkg.lib().mmrs_paged_attend_workspace_bytes
    assert need(4, 20, 48, 8) > 0 and need(0, 0, 1, 1) > 0
    for bad in ((-1, 1, 48, 8), (1025, 1, 48, 8), (1, -1, 48, 8), (1, 1, 48, 0), (1, 1, 47, 8), (1, 1, 17, 1), (1, 1, 4, 8)):
        assert need(*bad) == 0, bad
    assert pkg.lib().mmrs_paged_attend_status(None) == pkg.MMRS_ERR_ARG


def verify_args(**ch):
    a = dict(logits=P, type=0, vocab=1000, cu=P, num_seqs=2, rows=6, max_q=4, draft=P, probs=P, u=P, noise=P, temp=None, tokens=P,
             accepted=P, logprobs=P, ws=P, ws_bytes=1 << 40)
    a.update(ch)
    return (*a.values(), None)


@pytest.mark.parametrize("ch,name", [
    (dict(type=3), "UNSUPPORTED"), (dict(vocab=0), "ARG"), (dict(vocab=(1 << 20) + 1), "ARG"), (dict(num_seqs=-1), "ARG"),
    (dict(num_seqs=1025), "ARG"), (dict(rows=-1), "ARG"), (dict(rows=65537), "ARG"), (dict(max_q=0), "ARG"),
    (dict(max_q=65), "ARG"), (dict(cu=None), "ARG"), (dict(tokens=None), "ARG"), (dict(accepted=None), "ARG"),
    (dict(logits=None), "ARG"), (dict(noise=None), "ARG"), (dict(draft=None), "ARG"), (dict(u=None), "ARG"),
    (dict(ws=None), "ARG"), (dict(ws=P + 16), "ARG"), (dict(ws_bytes=256), "ARG"),
])
def test_verify(pkg, ch, name):
    assert pkg.lib().mmrs_verify_drafts(*verify_args(**ch)) == getattr(pkg, "MMRS_ERR_" + name)


def test_verify_of_nothing_and_workspace(pkg):
    lib = pkg.lib()
    assert lib.mmrs_verify_drafts(*verify_args(num_seqs=0, rows=0, cu=None)) == pkg.MMRS_OK
    assert lib.mmrs_verify_workspace_bytes(3, 12) > 0
    for bad in ((-1, 1), (1025, 1), (1, -1), (1, 65537)):
        assert lib.mmrs_verify_workspace_bytes(*bad) == 0
    assert lib.mmrs_verify_workspace_status(None) == pkg.MMRS_ERR_ARG


def test_python_checks(pkg):
    """The wrappers' own checks, on CPU tensors."""
    import torch
    k = torch.zeros(2, 2, 16, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(2, 2)
    make = pkg.PagedKvCache.from_tensors
    assert make(k, k, s, s).page_size == 16
    for bad in ((k.view(torch.uint8), k, s, s), (k, k[:1], s, s), (k, k, s.double(), s), (k, k, s, s[:1]),
                (k[:, :, ::2], k[:, :, ::2], s, s)):
        with pytest.raises(pkg.MoeError):
            make(*bad)
    with pytest.raises(pkg.MoeError):
        pkg.PagedKvCache(2, "cpu", kv_heads=2, page_size=24)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(pkg.MoeError):  # not on the device
        pkg.PagedBatch(i32, i32[:2], torch.zeros(2, 1, dtype=torch.int32), max_q=1, max_len=1)
    with pytest.raises(pkg.MoeError):
        pkg.DraftVerifier(100, "cpu", max_seqs=0, max_rows=1, max_q=1)


def test_python_calls_refuse_tensors_that_are_not_on_the_gpu(pkg):
    """A raw pointer to host memory would fault the device: the wrappers ask before they call."""
    import types

    import torch
    i32 = torch.zeros(3, dtype=torch.int32)
    batch = types.SimpleNamespace(t=(i32, i32[:2], torch.zeros(2, 1, dtype=torch.int32)), num_seqs=2)
    cache = pkg.PagedKvCache(2, "cpu", kv_heads=2, page_size=16)
    q, k, rope = torch.zeros(2, 12, 128), torch.zeros(2, 2, 128), torch.zeros(16, 32)
    with pytest.raises(pkg.MoeError, match="GPU"):
        cache.append(batch, q, k, k, rope, rope)
    with pytest.raises(pkg.MoeError, match="GPU"):
        cache.attend(batch, q.half())
    ver = pkg.DraftVerifier(100, "cpu", max_seqs=2, max_rows=4, max_q=2)
    with pytest.raises(pkg.MoeError, match="GPU"):
        ver.verify(torch.zeros(4, 100), i32, i32[:2], torch.zeros(2), torch.ones(2, 100))
