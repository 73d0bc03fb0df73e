"""What of `vcr_gaus_amd.optim`'s rarer calls needs no device."""
import copy
import ctypes as C
import gc
import pickle
import weakref
from array import array

import pytest
import torch

from vcr_gaus_amd import _lib
from vcr_gaus_amd.gaussian_model import FusedAdam, GaussianAdamW
from vcr_gaus_amd.optim import AdamW, decode8, encode8, rows8


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


def model_groups():
    """(as `GaussianModel` makes them, with a classifier)"""
    shapes = dict(xyz=(4, 3), f_dc=(4, 1, 3), opacity=(4, 1))
    groups = [dict(params=[P(*s)], lr=0.1, name=k) for k, s in shapes.items()]
    return groups + [dict(params=[P(2, 3)], lr=0.1, name="classifier.weight", aux=True), dict(params=[P(2)], lr=0.1, name="classifier.bias", aux=True)]


def state_of(shape, first=0.0, **other):
    n = int(torch.tensor(shape).prod())
    return dict(step=torch.tensor(7.0), exp_avg=torch.arange(first, first + n).view(shape), exp_avg_sq=torch.ones(shape), **other)


@pytest.mark.parametrize("of", ["exp_avg", "exp_avg_sq", "master"])
def test_moments_of_another_shape_are_refused(of):
    """As many values in another order: refused, and the optimizer stays as it was."""
    opt = AdamW([torch.nn.Parameter(torch.zeros(4, 3, dtype=torch.bfloat16))], master_weights=True)
    sd = opt.state_dict()
    sd["state"] = {0: state_of((4, 3), master=torch.zeros(4, 3))}
    opt.load_state_dict(sd)
    before = opt.state["0"]
    bad = copy.deepcopy(sd)
    bad["state"][0][of] = bad["state"][0][of].t()
    bad["param_groups"][0]["lr"] = 9.0
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(bad)
    assert opt.state["0"] is before and opt.param_groups[0]["lr"] == 1e-3


@pytest.mark.parametrize("cls", [GaussianAdamW, FusedAdam])
def test_model_optimizers_refuse_moments_of_another_shape(cls):
    opt = cls(model_groups())
    sd = dict(state={0: state_of((3, 4))}, param_groups=[dict(name="xyz", lr=0.5, params=[0])])
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(sd)
    sd["state"][0] = state_of((4, 3))
    opt.load_state_dict(sd)
    assert torch.equal(opt.state["xyz"]["exp_avg"], torch.arange(12.0).view(4, 3)) and opt.param_groups[0]["lr"] == 0.5


@pytest.mark.parametrize("cls", [GaussianAdamW, FusedAdam])
def test_model_optimizers_read_files_keyed_by_group_name(cls):
    """The older form: state by group name, the classifier's tensors by their own; groups that the file lacks keep rate and no state."""
    opt = cls(model_groups())
    sd = dict(state={"xyz": state_of((4, 3)), "classifier.bias": state_of((2,), 5.0), "gone": state_of((9,))},
              param_groups=[dict(name="xyz", lr=0.5), dict(name="f_dc", lr=0.25), dict(name="gone", lr=1.0)])
    opt.load_state_dict(sd)
    assert sorted(opt.state) == ["classifier.bias", "xyz"] and int(opt.state["xyz"]["step"]) == 7
    assert torch.equal(opt.state["xyz"]["exp_avg"], torch.arange(12.0).view(4, 3))
    assert torch.equal(opt.state["classifier.bias"]["exp_avg"], torch.tensor([5.0, 6.0]))
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.25, 0.1, 0.1, 0.1]
    sd["state"]["xyz"] = state_of((3, 4))
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(sd)


def test_the_kind_of_the_state_is_fixed():
    """Codes would be read as values, or the other way round."""
    opt = copy.deepcopy(AdamW([P(3)], state_bits=8, master_weights=True))
    assert opt.state_bits == 8 and opt.master_weights is True
    with pytest.raises(AttributeError):
        opt.state_bits = 32
    with pytest.raises(AttributeError):
        opt.master_weights = False


@pytest.mark.parametrize("kw", [dict(amsgrad=True), dict(maximize=True)])
def test_checkpoints_of_another_update_are_refused(kw):
    """torch.optim.AdamW's variants that this update does not have: not continued as something else without a word."""
    p = P(3)
    p.grad = torch.ones(3)
    ref = torch.optim.AdamW([dict(params=[p], name="xyz")], **kw)
    ref.step()
    for opt in (AdamW([p]), GaussianAdamW([dict(params=[p], name="xyz")])):
        with pytest.raises(ValueError, match=next(iter(kw))):
            opt.load_state_dict(ref.state_dict())
        assert opt.state == {}


def test_codes_and_values_that_do_not_fit_are_refused():
    """Before anything reaches a device: the kernels go by the number of codes alone."""
    def state(**other):
        st = {k: torch.zeros(300 if "scale" not in k else 2, dtype=torch.uint8) for k in
              ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
        st.update(other)
        return st

    x = torch.zeros(300)
    for k in state():
        n = state()[k].numel()
        for bad in (torch.zeros(n - 1, dtype=torch.uint8), torch.zeros(n), torch.zeros(2 * n, dtype=torch.uint8)[::2]):
            with pytest.raises(ValueError, match="exp_avg"):
                decode8(state(**{k: bad}))
            with pytest.raises(ValueError, match="exp_avg"):
                encode8(x, x, state(**{k: bad}))
    for bad in (x[:299], x.double(), torch.zeros(600)[::2], torch.zeros(0)):
        for m, v in ((bad, x), (x, bad)):
            with pytest.raises(ValueError, match="values of"):
                encode8(m, v, state())
    with pytest.raises(ValueError, match="HIP device"):
        encode8(x, x, state())
    with pytest.raises(ValueError, match="HIP device"):
        decode8(state())


def test_native_lists_find_shared_memory():
    native, x = _lib.tensor_list(), torch.zeros(100)
    far = torch.zeros(100)
    for tensors, want in (([], None), ([x], None), ([x, far], None), ([x, x], (0, 1)), ([x[:50], x[50:]], None), ([x[:51], far, x[50:]], (0, 2)),
                          ([x[10:20], x[30:40], x[:35]], (0, 2)), ([x, x[5:6], x[90:91]], (0, 1)), ([x[:0], x, x[50:50]], None),
                          ([x[20:40], x[:20].view(torch.bfloat16), x[40:].view(torch.uint8)], None), ([x[:21].view(torch.uint8), x[20:40]], (0, 1))):
        assert native.sharing(tensors) == want, want
        for k in range(len(tensors) + 1):
            assert native.sharing(tensors[:k], tensors[k:]) == want, want
    assert native.sharing() is None
    for bad in ((x,), [x, 1]):
        with pytest.raises(TypeError):
            native.sharing([x], bad)


@pytest.mark.parametrize("huge", [2 ** 63 - 1, 2 ** 62, 4096 * 4194303 + 1])
def test_c_entries_refuse_tensors_that_no_launch_can_hold(huge):
    """With a reason, and before anything reaches a device; the largest sizes overflow no sum on the way."""
    lib = _lib.load()
    word = lambda kind, *v: (lambda a: (a, a.buffer_info()[0]))(array(kind, v))  # noqa: E731
    (_n, numel), (_p, ptrs), (_k, kinds), (_g, group_of) = word("q", 8, huge, huge), word("Q", *[4096] * 3), word("i", 0, 0, 0), word("i", 0, 0, 0)
    groups = (_lib.VcrOptimGroup * 1)(_lib.VcrOptimGroup(1e-3, 0.9, 0.999, 1e-8, 0.0, None))
    step = _lib.VcrAdamWStep(ntensors=3, ngroups=1, state_bits=32, plan=4096, grads=ptrs, numel=numel, group_of=group_of, groups=groups)
    rec = (_lib.VcrOptimTensor * 3)()
    for r, n in zip(rec, (8, huge, huge)):
        r.p = r.m = r.v = r.step = 4096
        r.numel = n
    host = C.create_string_buffer(4096)
    assert lib.vcr_optim_plan_bytes(3, numel) == 0
    calls = [lambda: lib.vcr_adamw_step(C.byref(step), None), lambda: lib.vcr_optim_plan(3, rec, C.addressof(host), 4096),
             lambda: lib.vcr_moments8_decode(3, 4096, numel, ptrs, ptrs, 0, None), lambda: lib.vcr_moments8_encode(3, 4096, numel, ptrs, ptrs, None)]
    if huge > 2 ** 45:                                  # (the norm takes more: 16 384 elements a piece, 2^31 - 1 pieces)
        calls += [lambda: lib.vcr_grad_norm(3, ptrs, numel, kinds, 4096, 1 << 20, 1.0, 1.0, 0, 4096, None, None),
                  lambda: lib.vcr_clip_gradients(3, ptrs, numel, kinds, 4096, 1.0, None)]
        assert 0 < lib.vcr_grad_norm_partials(3, numel) < 10000
    for call in calls:
        _lib.load().vcr_adamw_step(None, None)          # (another error in between)
        assert call() == 1 and "tensor 1 with" in _lib.last_error() and "too large" in _lib.last_error()


def test_rows_of_codes_are_checked():
    lib = _lib.load()
    st = {k: torch.zeros((100, 3) if "scale" not in k else 2, dtype=torch.uint8) for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
    index = torch.zeros(5, dtype=torch.int32)
    for bad in (index.long(), index.view(5, 1), torch.zeros(10, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="index"):
            rows8([st], bad)
    for bad in (dict(st, exp_avg_sq=st["exp_avg_sq"].view(300)), dict(st, exp_avg=st["exp_avg"].view(3, 100))):
        with pytest.raises(ValueError, match="rows"):
            rows8([st, bad] if bad["exp_avg"].shape != (100, 3) else [bad], index)
    with pytest.raises(ValueError, match="exp_avg_scale"):
        rows8([dict(st, exp_avg_scale=torch.zeros(1, dtype=torch.uint8))], index)
    with pytest.raises(ValueError, match="HIP device"):
        rows8([st], index)
    arr = lambda width, **kw: (_lib.VcrRows8 * 1)(_lib.VcrRows8(width=width, **dict(  # noqa: E731
        dict.fromkeys(("m", "v", "m_scale", "v_scale", "m_out", "v_out", "m_scale_out", "v_scale_out"), 4096), **kw)))
    for args, msg in (((-1, None, 1, 1, 4096, None), "inconsistent"), ((1, None, 1, 1, 4096, None), "inconsistent"),
                      ((1, arr(3), -1, 1, 4096, None), "inconsistent"), ((1, arr(3), 1, 1, None, None), "inconsistent"),
                      ((1, arr(0), 1, 1, 4096, None), "width 0"), ((1, arr(3), 2 ** 62, 1, 4096, None), "width 3"),
                      ((1, arr(3), 1, 2 ** 34, 4096, None), "width 3"), ((1, arr(3, v=None), 1, 1, 4096, None), "pointer"),
                      ((1, arr(3, m_scale_out=None), 0, 1, 4096, None), "pointer")):
        assert lib.vcr_moments8_rows(*args) == 1 and msg in _lib.last_error(), (args, _lib.last_error())
    assert lib.vcr_moments8_rows(1, arr(3, m_out=None), 7, 0, None, None) == 0 and lib.vcr_moments8_rows(0, None, 0, 0, None, None) == 0
