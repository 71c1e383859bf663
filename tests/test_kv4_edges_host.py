"""Edges of the 4-bit cache's Python side, without a GPU: the library's calls are taken by a stand-in."""

import contextlib
import ctypes

import pytest
import torch

from tfimage import _lib, kernels as K, kv4


class OnGpu(torch.Tensor):
    """A CPU tensor that says it lies on CUDA device 3; nothing here follows its address."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    def get_device(self):
        return 3

    def new_empty(self, *a, **k):
        return OnGpu(torch.empty(*a, **{"dtype": self.dtype, **k}))


def gpu(*shape, dtype=torch.int32):
    return OnGpu(torch.zeros(shape, dtype=dtype))


@pytest.mark.parametrize("B,N", [(1, 0), (0, 4), (0, 0)])
def test_rotation_of_no_tokens(monkeypatch, B, N):
    """Empty tensors have null addresses."""
    monkeypatch.setattr(_lib, "launch", lambda index, fn, *args: _lib.check(fn(*args, None)))
    q, k = (OnGpu(torch.empty((B, N, h, 64), dtype=torch.bfloat16)) for h in (4, 2))
    out, k_out = K.rope_axes(q, k, OnGpu(torch.empty((N, 3))), (16, 24, 24), q_out=OnGpu(torch.empty_like(q)),
                             k_out=OnGpu(torch.empty_like(k)))
    assert out.shape == q.shape and k_out.shape == k.shape
    assert B or _lib.load().tfb_rope_axes(None, None, 4, None, None, 2, 2, B, 4, 60, (ctypes.c_int64 * 12)(), None, 0, 0, 3, 1,
                                          (ctypes.c_int * 1)(16), 1e4, None, None, 1e-6, 1, None) == 1   # D is still looked at


@pytest.fixture
def calls(monkeypatch):
    """The library's calls as (name, device that was current); device 0 is current outside of them."""
    seen, current = [], [0]

    class Library:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[0], args))
                return 4096 if name.endswith("_ws") else 0
            return call

    @contextlib.contextmanager
    def device(index):
        old, current[0] = current[0], index
        yield
        current[0] = old

    monkeypatch.setattr(_lib, "load", lambda: Library())
    monkeypatch.setattr(_lib, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    return seen


def cache_on_gpu():
    new = lambda n: gpu(4, 2, 64, n, dtype=torch.uint8)   # noqa: E731
    return kv4.Kv4Cache(new(64), new(8), new(64), new(8), 0.01, 0.02)


def test_workspace_is_asked_for_on_the_caches_device(calls):
    """The size goes by the SMs of the device that runs the call, which need not be the current one."""
    q = gpu(4, 4, 128, dtype=torch.bfloat16)
    kv4.attention(q, cache_on_gpu(), gpu(2, 3), gpu(2), out=gpu(4, 4, 128, dtype=torch.bfloat16))
    assert [(name, dev) for name, dev, _ in calls] == [("tfb_kv4_attention_ws", 3), ("tfb_kv4_attention", 3)]
    assert calls[1][2][-1] == 1003                       # its current stream


@pytest.mark.parametrize("name", ["k_codes", "k_sf", "v_codes", "v_sf", "k_global", "v_global", "pages", "heads", "page_size", "dim"])
def test_a_cache_cannot_be_changed_behind_its_calls(name):
    """The calls use the constructor's addresses and factors: assigning others would be silently ignored, or leave them on
    freed memory."""
    cache = kv4.Kv4Cache.empty(4, 64, 2, 128, 0.01, 0.02, device="cpu")
    old = getattr(cache, name)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.cat([old, old]) if isinstance(old, torch.Tensor) else 2 * old)
    assert getattr(cache, name) is old
