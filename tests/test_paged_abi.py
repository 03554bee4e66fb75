"""CPU checks of the paged cache's C entry points: null arguments are refused with a status."""
import ctypes
import types

import pytest
import torch

import ssdllm


def test_null_arguments_are_refused():
    L = ssdllm.lib()
    h = ctypes.c_void_p()
    assert L.ssd_kv_create_paged(None, 4, 16, 2, 64, ssdllm.F16, ctypes.byref(h)) == 1
    assert not h.value
    assert L.ssd_rope_table(None, 64, 1e4, 4, None, None) == 1
    assert L.ssd_paged_append(None, None, None, 0, 0, None, 0, None, 0, 0, None, None, 1e-5, None, 0, 0, 0,
                              None, None, None, 0, 0, None, 0, None) == 1
    assert L.ssd_paged_read(None, None, 0, None, None, None, 0, 0, 0, None, 0, None, 0, None) == 1
    n = ctypes.c_size_t()
    assert L.ssd_paged_attention_workspace(None, None, ctypes.byref(n)) == 1
    assert L.ssd_paged_attention(None, None, None, 0, 1, 0, None, None, None, 0, 0, 0.0, 0, None, 0, None, 0,
                                 None) == 1
    assert b"null" in L.ssd_last_error()


class OnGpu:
    """A tensor's looks, on any GPU."""

    def __init__(self, gpu, *shape, dtype=torch.float32):
        self.gpu, self.t, self.dtype = gpu, torch.empty(shape, dtype=dtype, device="meta"), dtype
        self.shape, self.device, self.is_cuda = self.t.shape, torch.device("cuda", gpu), True

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.gpu

    def data_ptr(self):
        return 4096


class Calls:
    """The library's entry points, noting their arguments."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        return lambda *a: self.made.append((name, a)) or 0


@pytest.fixture
def cache(monkeypatch):
    """A cache on the second GPU, its calls, and the streams that were current on each."""
    calls = Calls()
    monkeypatch.setattr(ssdllm, "lib", lambda: calls)
    monkeypatch.setattr(ssdllm, "_raw_stream", lambda device: 7000 + device)
    kv = ssdllm.PagedKvCache.__new__(ssdllm.PagedKvCache)
    kv.h, kv.torch, kv.ctx = None, torch, types.SimpleNamespace(h=None, device=1)
    kv.n_head_kv, kv.head_dim = 2, 64
    return kv, calls


def test_tensors_and_streams_are_those_of_the_contexts_gpu(cache):
    kv, calls = cache
    rows = lambda gpu=1: OnGpu(gpu, 3, 128)  # noqa: E731
    ints = lambda *shape: OnGpu(1, *shape, dtype=torch.int32)  # noqa: E731
    good = {"append": dict(k=rows(), v=rows(), pos=ints(3), table=ints(3, 4), seq=ints(3), q=rows(), q_out=rows(),
                           q_norm=OnGpu(1, 64), k_norm=OnGpu(1, 64), rope=OnGpu(1, 9, 32, 2)),
            "read": dict(pos=ints(3), table=ints(3, 4), k_out=rows(), v_out=rows(), seq=ints(3)),
            "attention": dict(q=rows(), length=ints(3), table=ints(3, 4), out=rows(),
                              workspace=OnGpu(1, 64, dtype=torch.uint8), seq=ints(3))}
    for name, args in good.items():
        getattr(kv, name)(**args)
        assert calls.made.pop()[1][-1] == 7001
        for which, t in args.items():
            with pytest.raises(ssdllm.SsdError) as e:
                getattr(kv, name)(**{**args, which: OnGpu(0, *t.shape, dtype=t.dtype)})
            assert e.value.status == 1 and not calls.made, (name, which)
    ssdllm.rope_table(kv.ctx, 64, 1e4, 9, OnGpu(1, 9, 32, 2))
    assert calls.made.pop()[1][-1] == 7001
    with pytest.raises(ssdllm.SsdError):
        ssdllm.rope_table(kv.ctx, 64, 1e4, 9, OnGpu(0, 9, 32, 2))
