"""What of `vcr_gaus_amd.optim` needs no device: arguments, state dictionaries, refusals of the C entries, the 8-bit format's arithmetic."""
import ctypes as C
from array import array

import numpy as np
import pytest
import torch

from tests import optim_reference as R
from vcr_gaus_amd import _lib
from vcr_gaus_amd.optim import AdamW, clip_grad_norm_, grad_norm


def P(*shape):
    return torch.nn.Parameter(torch.zeros(*shape))


@pytest.mark.parametrize("kw, msg", [
    (dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "out of range"), (dict(betas=(1.0, 0.9)), "out of range"),
    (dict(betas=(0.9, -0.1)), "out of range"), (dict(eps=-1e-8), "out of range"), (dict(eps=1e-40), "out of range"),
    (dict(weight_decay=-0.1), "out of range"), (dict(lr=float("nan")), "out of range"), (dict(lr=torch.zeros(2)), "one float32 element")])
def test_constructor_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        AdamW([P(3)], **kw)


def test_constructor_refuses_lists():
    p = P(2)
    with pytest.raises(ValueError, match="no parameters"):
        AdamW([])
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, p])
    with pytest.raises(TypeError, match="among the parameters"):
        AdamW([p, 3])
    with pytest.raises(TypeError, match="dictionaries"):
        AdamW([dict(params=[p]), p])
    opt = AdamW([dict(params=[P(2)], name="a"), dict(params=[P(3)], name="a")])
    with pytest.raises(ValueError, match="not unique"):
        opt.state_dict()


def test_host_tensors_are_refused_where_the_kernels_would_read_them():
    p = P(4)
    p.grad = torch.ones(4)
    with pytest.raises((ValueError, RuntimeError, AssertionError)):
        AdamW([p]).step()
    with pytest.raises(ValueError, match="HIP device"):
        grad_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="HIP device"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="no tensors"):
        grad_norm([])
    with pytest.raises(TypeError, match="not a tensor"):
        grad_norm([1.0])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        grad_norm([torch.ones(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="must be > 0"):
        clip_grad_norm_([p], 0.0)
    with pytest.raises(ValueError, match="no parameter has a gradient"):
        clip_grad_norm_([P(1)], 1.0)


def test_no_gradient_is_no_step():
    opt = AdamW([P(4)])
    assert opt.step() is None and opt.step(max_norm=1.0) is None and opt.state == {}
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)


def test_groups_defaults_and_keys():
    a, b, c = P(2), P(3), P(4)
    opt = AdamW([dict(params=[a, b], lr=0.5), dict(params=c, name="head", weight_decay=0.0)], lr=0.1, betas=(0.8, 0.9), weight_decay=0.2)
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.1] and [g["weight_decay"] for g in opt.param_groups] == [0.2, 0.0]
    assert opt._keys() == ["0.0", "0.1", "head"]


def test_state_dictionary_layout_is_torchs():
    a, b = P(2, 3), P(5)
    opt = AdamW([dict(params=[a], lr=0.5), dict(params=[b])], lr=0.1)
    sd = opt.state_dict()
    ref = torch.optim.AdamW([dict(params=[a], lr=0.5), dict(params=[b])], lr=0.1)
    assert sd["state"] == {} and [g["params"] for g in sd["param_groups"]] == [[0], [1]]
    assert set(ref.state_dict()["param_groups"][0]) <= set(sd["param_groups"][0])
    for p in (a, b):
        p.grad = torch.randn_like(p)
    ref.step()
    opt.load_state_dict(ref.state_dict())
    assert opt.state["0"]["step"].dtype == torch.int32 and int(opt.state["1"]["step"]) == 1
    assert torch.equal(opt.state["0"]["exp_avg"], ref.state[a]["exp_avg"])
    ref2 = torch.optim.AdamW([dict(params=[a], lr=0.5), dict(params=[b])], lr=0.1)
    ref2.load_state_dict(opt.state_dict())
    assert torch.equal(ref2.state[b]["exp_avg_sq"], ref.state[b]["exp_avg_sq"]) and float(ref2.state[b]["step"]) == 1.0
    with pytest.raises(ValueError, match="groups saved"):
        AdamW([a, b]).load_state_dict(sd)
    with pytest.raises(ValueError, match="tensors saved"):
        AdamW([dict(params=[a, b]), dict(params=[P(1)])]).load_state_dict(sd)
    bad = ref.state_dict()
    bad["state"][0]["exp_avg"] = torch.zeros(7)
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(bad)


def test_replacing_state_makes_the_optimizer_look_again():
    opt = AdamW([P(3)])
    opt.state = {"0": dict(step=torch.zeros((), dtype=torch.int32))}
    for change in (lambda: opt.state.update(a={}), lambda: opt.state.pop("a"), lambda: opt.state["0"].__setitem__("exp_avg", torch.zeros(3)),
                   lambda: opt.state["0"].setdefault("exp_avg_sq", torch.zeros(3)), lambda: setattr(opt, "state", {})):
        opt._plan = "built"
        change()
        assert opt._plan is None


def test_copies_and_added_groups():
    import copy
    import pickle
    opt = AdamW([P(3)], lr=0.5, state_bits=8)
    opt.state = {"0": dict(step=torch.zeros((), dtype=torch.int32))}
    opt._plan = lambda: None                            # (something that cannot be copied)
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert twin._plan is None and twin.state_bits == 8 and int(twin.state["0"]["step"]) == 0
        twin._plan = "built"
        twin.state["0"]["step"] = torch.ones((), dtype=torch.int32)
        assert twin._plan is None and int(opt.state["0"]["step"]) == 0
    q = P(4)
    opt.add_param_group(dict(params=q, name="late", lr=0.1))
    assert opt._keys() == ["0", "late"] and opt.param_groups[1]["weight_decay"] == 1e-2
    for bad in (dict(params=[q]), dict(params=[P(1)], lr=-1.0), dict(lr=1.0)):
        with pytest.raises((ValueError, TypeError)):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 2


# ---- C entries: refused before anything reaches a device -----------------------------------------------------------------
def _words(kind, values):
    a = array(kind, values)
    return a, a.buffer_info()[0]


def _step_args(**kw):
    n, numel = _words("q", [8])
    g, group_of = _words("i", [0])
    q, grads = _words("Q", [4096])
    groups = (_lib.VcrOptimGroup * 1)(_lib.VcrOptimGroup(1e-3, 0.9, 0.999, 1e-8, 0.0, None))
    a = dict(ntensors=1, ngroups=1, param_type=0, state_bits=32, plan=4096, grads=grads, numel=numel, group_of=group_of, groups=groups)
    a.update(kw)
    return _lib.VcrAdamWStep(**a), (n, g, q, groups)


def test_c_step_refuses_and_says_why():
    lib = _lib.load()
    assert lib.vcr_adamw_step(None, None) == 1 and "NULL" in _lib.last_error()
    bad_beta = (_lib.VcrOptimGroup * 1)(_lib.VcrOptimGroup(1e-3, 1.0, 0.999, 1e-8, 0.0, None))
    neg, neg_at = _words("q", [-1])
    far, far_at = _words("i", [3])
    for kw, msg in [(dict(state_bits=16), "inconsistent"), (dict(param_type=3), "inconsistent"), (dict(param_type=-1), "inconsistent"),
                    (dict(grads=None), "inconsistent"), (dict(ngroups=0), "inconsistent"), (dict(plan=None), "plan"),
                    (dict(numel=None), "numel"), (dict(masters=1), "inconsistent"), (dict(groups=bad_beta), "beta1"),
                    (dict(numel=neg_at), "numel -1"), (dict(group_of=far_at), "group 3 of 1"), (dict(ntensors=-2), "plan or numel")]:
        a, keep = _step_args(**kw)
        assert lib.vcr_adamw_step(C.byref(a), None) == 1, kw
        assert msg in _lib.last_error(), (kw, _lib.last_error())
    a, keep = _step_args(ntensors=0)
    assert lib.vcr_adamw_step(C.byref(a), None) == 0


def test_c_lists_and_plans_refuse():
    lib = _lib.load()
    n, numel = _words("q", [8, 4])
    p, ptrs = _words("Q", [4096, 0])
    k, kinds = _words("i", [0, 1])
    k9, kinds9 = _words("i", [0, 9])
    assert lib.vcr_grad_norm(2, ptrs, numel, kinds, 4096, 64, 1.0, 0.0, 0, 4096, None, None) == 1 and "tensor 1" in _lib.last_error()
    assert lib.vcr_grad_norm(1, ptrs, numel, kinds, None, 64, 1.0, 0.0, 0, 4096, None, None) == 1 and "partials" in _lib.last_error()
    assert lib.vcr_grad_norm(1, ptrs, numel, kinds, 4096, 64, 1.0, 0.0, 0, None, None, None) == 1
    assert lib.vcr_grad_norm(1, ptrs, numel, kinds, 4096, 0, 1.0, 0.0, 0, 4096, None, None) == 1 and "too little" in _lib.last_error()
    assert lib.vcr_grad_norm(1, ptrs, numel, kinds, 4096, 64, 1.0, 0.0, 0, 4096, 4096, None) == 1 and "max_norm" in _lib.last_error()
    assert lib.vcr_grad_norm(2, ptrs, numel, kinds9, 4096, 64, 1.0, 0.0, 0, 4096, None, None) == 1 and "type 9" in _lib.last_error()
    assert lib.vcr_clip_gradients(1, ptrs, numel, kinds, None, 1.0, None) == 1
    assert lib.vcr_clip_gradients(1, ptrs, numel, kinds, 4096, 0.0, None) == 1 and "max_norm" in _lib.last_error()
    assert lib.vcr_moments8_decode(1, None, numel, ptrs, ptrs, 0, None) == 1
    assert lib.vcr_moments8_decode(1, 4096, numel, ptrs, ptrs, 5, None) == 1
    assert lib.vcr_moments8_encode(2, 4096, numel, ptrs, ptrs, None) == 1 and "missing" in _lib.last_error()
    rec = (_lib.VcrOptimTensor * 1)()
    rec[0].numel = 8
    host = C.create_string_buffer(4096)
    assert lib.vcr_optim_plan(1, rec, C.addressof(host), 4096) == 1 and "pointer missing" in _lib.last_error()
    rec[0].p = rec[0].m = rec[0].v = rec[0].step = 4096
    assert lib.vcr_optim_plan(1, rec, C.addressof(host), 16) == 1 and "16 bytes" in _lib.last_error()
    size = lib.vcr_optim_plan_bytes(1, numel)
    assert 0 < size <= 4096 and lib.vcr_optim_plan(1, rec, C.addressof(host), size) == 0
    rec[0].m_scale = 4096
    assert lib.vcr_optim_plan(1, rec, C.addressof(host), size) == 1
    assert lib.vcr_optim_plan_bytes(0, numel) == 0 and lib.vcr_optim_plan_bytes(1, None) == 0


def test_norm_scratch_is_enough_for_any_mix_of_types():
    """One partial sum per workgroup, at most 1 024 workgroups a launch, at most 192 tensors of one type a launch."""
    lib = _lib.load()
    rng = np.random.default_rng(3)
    for trial in range(50):
        n = int(rng.integers(1, 900))
        numel = rng.integers(0, 10, n) * rng.choice([1, 1000, 10 ** 7], n)
        kinds = rng.integers(0, 3, n)
        need = 0
        for k in range(3):
            mine = [int(x) for x in numel[kinds == k] if x > 0]
            for i in range(0, len(mine), 192):
                need += min(1024, sum(-(-x // 16384) for x in mine[i:i + 192]))
        a, at = _words("q", [int(x) for x in numel])
        assert lib.vcr_grad_norm_partials(n, at) >= need


# ---- the 8-bit format ------------------------------------------------------------------------------------------------------
def test_codes_of_the_reference_round_trip():
    """Every code under every block exponent stands for a value whose nearest code it is (the largest value of the block is kept in
    the top binade, as in a stored block)."""
    for signed, top in ((True, 14), (False, 30)):
        for s in (1, 2, 14, 31, 90, 127, 200, 254):
            codes = np.arange(256, dtype=np.uint8)
            if signed:
                codes = codes[(codes & 0x7F) < 0x78]
            else:
                codes = codes[codes < 0xF8]
            x = R.decode(codes, np.array([s], np.uint8), signed)
            c, sc = R.encode(x, R.nearest, signed)
            back = R.decode(c, sc, signed)
            live = np.abs(x) > 0
            if s > 30:
                assert sc[0] == s
                assert np.array_equal(back, x)
            else:                                     # (near the bottom of fp32 the values themselves are rounded)
                assert np.all(np.abs(back - x)[live] <= np.abs(x)[live] * 2.0 ** -4 + 2.0 ** -149)


def test_stochastic_rounding_of_the_reference_is_unbiased():
    """A value a third of the way between two codes goes up in a third of the cases: 10^6 draws, five standard deviations."""
    n = 1 << 20
    for signed, shift in ((True, np.uint64(16)), (False, np.uint64(0))):
        x = np.full(n, F := np.float32((1 + 1 / 24) * 2.0 ** -3), np.float32)
        x[::256] = 1.0                                # (the block's largest value)
        w = R.words(7, 11, 3, n)
        r = ((w >> shift & np.uint64(65535)) * np.uint64(16) + np.uint64(8)).astype(np.int64)
        c, s = R.encode(x, r, signed)
        v = R.decode(c, s, signed).astype(np.float64)[x == F]
        step = 2.0 ** -6
        assert set(np.unique(v)) == {2.0 ** -3, 2.0 ** -3 + step}
        sigma = step * np.sqrt(2 / 9 / v.size)
        assert abs(v.mean() - float(F)) < 5 * sigma + step * 2.0 ** -16


def test_random_words_do_not_repeat_between_steps_tensors_and_blocks():
    base = R.words(1, 1, 0, 4096)
    for other in (R.words(2, 1, 0, 4096), R.words(1, 2, 0, 4096), R.words(1, 1, 1, 4096)):
        assert np.mean(base == other) < 0.01 and abs(np.corrcoef(base.astype(float), other.astype(float))[0, 1]) < 0.1
    assert np.unique(R.words(1, 1, 0, 1 << 16)).size > (1 << 16) * 0.99


# ---- native lists, on the host -----------------------------------------------------------------------------------------------
def test_native_lists_leave_host_tensors_to_the_checks():
    native = _lib.tensor_list()
    p = P(3)
    p.grad = torch.ones(3)
    assert native.words([p]) is None and native.words([]) is None and native.words(p) is None and native.words([None]) is None
    assert native.gradients([p], None) is None and native.gradients([], None) is None
    before = p._version
    native.changed([p, p.grad, 3], None)
    assert p._version == before + 1
    native.changed([p, p.grad], bytes(8) + b"\1" + bytes(7))
    assert p._version == before + 1 and p.grad._version == 2
    with torch.inference_mode():
        q = torch.ones(2)
    native.changed([q], None)
    with pytest.raises(TypeError):
        native.changed((p,), None)
