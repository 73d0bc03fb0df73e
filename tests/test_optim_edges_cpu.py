"""What of `vcr_gaus_amd.optim`'s rarer calls needs no device."""
import copy
import gc
import pickle
import weakref

import pytest
import torch

from vcr_gaus_amd import _lib
from vcr_gaus_amd.optim import AdamW


def P(*shape):
    return torch.nn.Parameter(torch.zeros(*shape))


@pytest.fixture
def no_collector():
    gc.collect()
    gc.disable()
    yield
    gc.enable()


def test_an_optimizer_goes_with_its_last_reference(no_collector):
    """No reference cycle: optimizer, parameters and moments are freed without the collector; a state dictionary that outlives its
    optimizer stays usable."""
    p = P(3)
    opt = AdamW([p])
    opt.state = {"0": dict(step=torch.zeros((), dtype=torch.int32), exp_avg=torch.zeros(3), exp_avg_sq=torch.zeros(3))}
    twin = copy.deepcopy(opt)
    again = pickle.loads(pickle.dumps(opt))
    seen = [weakref.ref(x) for x in (opt, p, opt.state["0"]["exp_avg"], twin, twin.param_groups[0]["params"][0], again)]
    kept = opt.state
    del opt, p, twin, again
    assert [r() is None for r in seen] == [True, True, False, True, True, True]
    kept["1"] = {}
    kept["0"]["exp_avg"] = torch.ones(3)
    assert list(kept) == ["0", "1"] and seen[2]() is None


def test_native_lists_know_a_tensors_memory():
    """`memory` / `in_place`: another storage, size, type or layout under the same object is seen, another value is not."""
    native = _lib.tensor_list()
    a, b = torch.zeros(6), torch.zeros((), dtype=torch.int32)
    known = native.memory([a, b])
    assert native.in_place([a, b], known) and not native.in_place([a], known) and not native.in_place([b, a], known)
    a.fill_(3.0)
    assert native.in_place([a, b], known)
    keep = a.data
    for other in (a.data.clone(), a.data[:5], a.data.view(2, 3).t()):
        a.data = other
        assert not native.in_place([a, b], known)
    a.data = keep
    assert native.in_place([a, b], known) and native.memory([]) == b"" and native.in_place([], b"")
    for bad in ((a,), [a, 1]):
        with pytest.raises(TypeError):
            native.memory(bad)
    assert not native.in_place([a, 1], known)
    with pytest.raises(TypeError):
        native.in_place((a, b), known)
