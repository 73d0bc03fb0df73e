"""What of `vcr_gaus_amd.optim`'s rarer calls needs no device."""
import copy
import gc
import pickle
import weakref

import pytest
import torch

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
