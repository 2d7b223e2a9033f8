"""Calls for tensors of a GPU that is not the current one are launched on the tensors' GPU.  Without a GPU: tensors
that say they lie on one, a runtime that only notes which GPU was current, and no library call."""
from __future__ import annotations

import contextlib
import types

import pytest
import torch


@pytest.fixture
def seen(pkg, monkeypatch):
    """(GPU that was current, name) of every library call; GPU 0 is current, the tensors lie on GPU 1."""
    calls, state = [], types.SimpleNamespace(gpu=0)
    real = pkg.lib()

    @contextlib.contextmanager
    def device(index):
        was, state.gpu = state.gpu, index
        yield
        state.gpu = was

    class Lib:
        def __getattr__(self, name):
            if not name.endswith(("append", "attend", "verify_drafts", "verify_drafts_n")):
                return getattr(real, name)
            return lambda *a: calls.append((state.gpu, name)) or 0

    class On1(torch.Tensor):
        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state.gpu)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(pkg, "lib", Lib)
    on = lambda t: t.as_subclass(On1)  # noqa: E731
    return types.SimpleNamespace(calls=calls, on=on, state=state)


STREAM = types.SimpleNamespace(cuda_stream=5)


def test_append_and_attend(pkg, seen):
    cache = pkg.PagedKvCache(2, "cpu", kv_heads=2, page_size=16)
    cache.device_index = 1
    table = seen.on(torch.zeros(2, 1, dtype=torch.int32))
    batch = types.SimpleNamespace(t=(None, seen.on(torch.zeros(2, dtype=torch.int32)), table), num_seqs=2,
                                  bind=lambda cache, n: None)
    q, k, rope = seen.on(torch.zeros(2, 12, 128)), seen.on(torch.zeros(2, 2, 128)), seen.on(torch.zeros(16, 32))
    q16 = seen.on(torch.zeros(2, 12, 128, dtype=torch.float16))
    cache.ws, cache._ws_ptr, cache._ws_bytes = torch.zeros(1 << 26, dtype=torch.uint8), 0, 1 << 26
    assert cache.append(batch, q, k, k, rope, rope, q_out=q16, stream=STREAM) is q16
    assert cache.attend(batch, q16, out=q16, stream=STREAM) is q16
    assert seen.calls == [(1, "mmrs_paged_append"), (1, "mmrs_paged_attend")] and seen.state.gpu == 0


def test_verify(pkg, seen):
    ver = pkg.DraftVerifier(100, "cpu", max_seqs=2, max_rows=4, max_q=2)
    ver.tokens = seen.on(ver.tokens)
    i32 = seen.on(torch.tensor([0, 2, 4], dtype=torch.int32))
    ver.verify(seen.on(torch.zeros(4, 100)), i32, seen.on(i32[:2]), seen.on(torch.zeros(2)), seen.on(torch.ones(2, 100)),
               stream=STREAM)
    assert [gpu for gpu, _ in seen.calls] == [1] and seen.state.gpu == 0
