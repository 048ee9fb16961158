"""route_experts' host side without a GPU: what the library is handed, with its entry point replaced."""
import ctypes
import gc
import weakref

import pytest
import torch

from fleet import mk, routing


class OnDevice:
    """Logits [4, 64] that say they are on CUDA device 0."""
    shape, dtype, device = torch.Size((4, 64)), torch.float32, torch.device("cpu")

    def dim(self):
        return 2

    def stride(self, i=None):
        return (64, 1) if i is None else (64, 1)[i]

    def get_device(self):
        return 0

    def data_ptr(self):
        return 4096


class Handed:
    """The library's calls: what `during` made of each call's parameters (a copy of them)."""

    def __init__(self):
        self.calls = []
        self.during = lambda p: mk.MkRoute.from_buffer_copy(ctypes.string_at(p, ctypes.sizeof(mk.MkRoute)))

    def __call__(self, params, *_):
        self.calls.append(self.during(params))
        return 0


@pytest.fixture
def handed(monkeypatch):
    h = Handed()
    monkeypatch.setattr(mk, "entry", lambda name: (h, lambda: 0, lambda index: 0, None))
    routing._params.cache_clear()
    return h


def test_parameters_live_as_long_as_the_call(handed, monkeypatch):
    """Another thread may route with so many other parameters during a call that the cache drops this call's."""
    made = []

    class Watched(mk.MkRoute):
        def __init__(self, *a):
            super().__init__(*a)
            made.append(weakref.ref(self))
    monkeypatch.setattr(mk, "MkRoute", Watched)

    def others(params):
        for k in range(1, 400):
            routing._params(64, 1, 0, 1, 1, "max", "softmax", False, torch.float32, float(k))
        gc.collect()
        return made[0]() is not None
    handed.during = others
    routing.route_experts(OnDevice(), 6)
    assert handed.calls == [True]


def test_scaling_is_a_number_not_an_object(handed):
    """A tensor hashes by its identity: the call after it changed must not get the first one's value."""
    scaling = torch.tensor(2.0)
    routing.route_experts(OnDevice(), 6, scaling=scaling)
    scaling.fill_(3.0)
    routing.route_experts(OnDevice(), 6, scaling=scaling)
    assert [p.scaling for p in handed.calls] == [2.0, 3.0]


def test_counts_are_integers(handed):
    import numpy as np
    ids, weights = routing.route_experts(OnDevice(), np.int64(6), n_forced=torch.tensor(2), renormalize=np.bool_(True))
    assert ids.shape == weights.shape == (4, 8)
    assert (handed.calls[0].topk, handed.calls[0].n_forced, handed.calls[0].renormalize) == (6, 2, 1)
    with pytest.raises(TypeError):
        routing.route_experts(OnDevice(), 6.0)


def test_a_stream_of_another_device_is_refused():
    """It would otherwise be ignored: the call runs on its tensors' device, on that device's current stream."""
    from types import SimpleNamespace
    on = SimpleNamespace(device=torch.device("cuda", 0))
    with pytest.raises(ValueError):
        mk.on_stream(on, SimpleNamespace(cuda_stream=64, device=torch.device("cuda", 1)))
    for stream in (64, SimpleNamespace(cuda_stream=64, device=torch.device("cuda", 0))):
        with pytest.raises(mk.MkError):
            mk.on_stream(SimpleNamespace(device=torch.device("cpu")), stream)


def test_tensors_of_a_call_on_a_stream_are_recorded(monkeypatch):
    from types import SimpleNamespace
    dev, stream = torch.device("cuda", 0), SimpleNamespace(cuda_stream=64, device=torch.device("cuda", 0))
    seen = []
    t = lambda name, device=dev: SimpleNamespace(device=device, record_stream=lambda s: seen.append((name, s)))  # noqa: E731
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
    assert mk.on_stream(t("x"), stream, None, t("ids"), t("other", torch.device("cpu"))) is stream
    assert seen == [("x", stream), ("ids", stream)]
