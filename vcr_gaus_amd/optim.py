"""Optimizer operators over many tensors at once: `AdamW` (moments in 32 or in 8 bits), `grad_norm`, `clip_grad_norm_`.

They stand beside `gaussian_model.FusedAdam` (Adam on the Gaussian model's groups, fp32, at most 8 tensors a launch) for what that one
does not do: decoupled weight decay, any number of tensors of any size and alignment, fp32 / bf16 / fp16 parameters with or without
fp32 masters, clipping by the norm of all gradients without a host round trip, step counters that live on the device (a captured
step replays), and moments in a quarter of the memory.  The reference trains with torch.optim.Adam only
(`scene/gaussian_model.py:258`); the update is torch.optim.AdamW's.  All arithmetic runs in csrc/optim.hip; there is no fallback.
"""
import ctypes as C
import sys
import weakref
from array import array

import torch

from . import _lib
from ._lib import tensor_list as _native

BLOCK = 256                                    # elements that share the scale of an 8-bit moment
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# Lists of many tensors go to the library as arrays of words.  Ordinary lists (plain dense contiguous tensors of the supported types on
# one device) are turned into them in one native call: at 160 tensors the host's share of a call is what a user sees (a loop over the
# tensors took 94 us, attribute by attribute 41 us, the kernels 10).  Any other list is looked at here, tensor by tensor.


def _address(words):
    return words.buffer_info()[0]


def _on(dev, call, *args):
    """`call(*args)` with `dev` the current device: the library launches on the current device, whatever device the stream is of."""
    if torch.cuda.current_device() == dev.index:
        return call(*args)
    with torch.cuda.device(dev):
        return call(*args)


def _check_list(tensors, what):
    """The types and the device of a list; every tensor dense, of a supported type and on the device of the first."""
    for k, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}[{k}] is a {type(t).__name__}, not a tensor")
        if t.dtype not in _TYPES:
            raise ValueError(f"{what}[{k}] has type {t.dtype}: float32, bfloat16 or float16 are supported")
        if not t.is_cuda or t.layout != torch.strided:
            raise ValueError(f"{what}[{k}] is not a dense tensor on a HIP device")
        if t.device != tensors[0].device:
            raise ValueError(f"{what}[{k}] is on {t.device}, {what}[0] on {tensors[0].device}")
    return [t.dtype for t in tensors], tensors[0].device if tensors else None


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _dense(tensors, what):
    """The tensors, contiguous and stored as they are read."""
    try:
        return [t if t.is_contiguous() and not t.is_neg() else t.detach().resolve_neg().contiguous() for t in tensors]
    except (RuntimeError, NotImplementedError) as e:          # (layouts that have no strides)
        raise ValueError(f"{what}: dense tensors are needed: {e}") from None


class _List:
    """Tensors as the library takes them: how many, addresses, sizes, types (`args`), on `device`.  `work`: the tensors that were
    listed, dense copies where the given ones are not dense; `holds`: what the addresses are of."""
    __slots__ = ("work", "device", "args", "holds")

    def __init__(self, tensors, what, where):
        n, found = len(tensors), _native().words(tensors)
        if found is not None:
            index, blob, at = found
            self.work, self.device, self.args, self.holds = tensors, tensors[0].device, (n, at, at + 8 * n, at + 16 * n), blob
            return
        dtypes, self.device = _check_list(tensors, what)
        self.work = _dense(tensors, where)
        self.holds = (array("Q", [t.data_ptr() for t in self.work]), array("q", [t.numel() for t in self.work]),
                      array("i", [_TYPES[d] for d in dtypes]))
        self.args = (n, *map(_address, self.holds))


def _norm(args, out, stream, again=False, grad_scale=1.0, max_norm=0.0, clip=False):
    """Launches the norm of the listed tensors into `out`; -> with `clip` the buffer whose first 8 bytes are the clipped step's factor.
    `again`: the tensors are read again right behind.
    The scratch belongs to this call (allocated on the current stream): two captured calls share nothing."""
    lib = _lib.load()
    room = lib.vcr_grad_norm_partials(args[0], args[2])
    buffer = torch.empty(room + 1, dtype=torch.float64, device=out.device)
    at = buffer.data_ptr()
    _lib.check(lib.vcr_grad_norm(*args, at + 8, room, grad_scale, max_norm, int(again), out.data_ptr(), at if clip else None, stream))
    return buffer


def grad_norm(tensors, out=None):
    """2-norm over all elements of all `tensors` (a list, or one tensor; float32 / bfloat16 / float16, mixed as they come) as a 0-dim
    float32 tensor on their device.  Sums in 64 bits in a fixed order: the same result on every run; NaN or infinity anywhere gives
    NaN or infinity.  No tensors: an error, as there is no device to put the result on -- unless `out` is given."""
    words = _List([tensors] if isinstance(tensors, torch.Tensor) else list(tensors), "tensors", "grad_norm")
    dev, own = words.device, out is None
    if own:
        if dev is None:
            raise ValueError("grad_norm: no tensors and no `out`")
        out = torch.empty((), device=dev)
    elif out.dtype != torch.float32 or out.numel() != 1 or not out.is_cuda or dev not in (None, out.device):
        raise ValueError("grad_norm: `out` must be one float32 element on the tensors' device")
    dev = out.device
    _on(dev, _norm, words.args, out, _stream(dev.index))
    if not own:
        _native().changed([out], None)
    return out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)), norm their 2-norm over all; -> norm (a 0-dim
    float32 tensor; nothing waits for it).  For optimizers that take gradients as they are; `AdamW.step(max_norm=...)` applies the
    factor inside the update instead, without writing the gradients again.  Gradients must not share memory, with each other or (expanded
    ones) with themselves."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = _positive(max_norm, "max_norm")
    grads = [p.grad for p in parameters]
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("clip_grad_norm_: no parameter has a gradient")
    if len(set(map(id, grads))) != len(grads):
        raise ValueError("clip_grad_norm_: a gradient appears twice")
    words = _List(grads, "gradients", "clip_grad_norm_")
    if words.work is not grads and any(n > 1 and s == 0 for g in grads for n, s in zip(g.shape, g.stride())):
        raise ValueError("clip_grad_norm_: an expanded gradient, whose elements share memory, cannot be scaled in place")
    twice = _native().sharing(words.work)
    if twice:
        raise ValueError(f"clip_grad_norm_: gradients {twice[0]} and {twice[1]} share memory")
    dev = words.device
    norm, stream = torch.empty((), device=dev), _stream(dev.index)

    def both():
        _norm(words.args, norm, stream, True)
        _lib.check(_lib.load().vcr_clip_gradients(*words.args, norm.data_ptr(), max_norm, stream))

    _on(dev, both)
    _native().changed(grads, None)
    if words.work is not grads:
        for g, w in zip(grads, words.work):
            if g is not w:
                g.copy_(w)
    return norm


def _positive(x, what):
    x = float(x)
    if not x > 0.0:
        raise ValueError(f"{what} = {x}: must be > 0")
    return x


class _Watched(dict):
    """A dictionary of the optimizer's state: an entry that is replaced, added or removed makes the optimizer look at its tensors anew
    (their addresses are on the device).  Values may be changed in place freely.  The optimizer is held weakly: with what it trains and
    its moments it goes when its last user lets go of it, not when the cyclic collector runs."""
    __slots__ = ("_owner",)

    def __init__(self, owner, items=()):
        dict.__init__(self, items)
        self._owner = weakref.ref(owner)

    def _touch(name):
        def method(self, *a, **k):
            owner = self._owner()
            if owner is not None:
                owner._plan = None
            return getattr(dict, name)(self, *a, **k)
        method.__name__ = name
        return method

    for _n in ("__setitem__", "__delitem__", "pop", "popitem", "clear", "update", "setdefault", "__ior__"):
        locals()[_n] = _touch(_n)
    del _n, _touch

    def __reduce__(self):
        return dict, (dict(self),)


class _Bucket:
    """The tensors of one type: their plan on the device and what a call needs of them on the host."""
    __slots__ = ("type", "at", "numels", "kinds", "group_of", "plan", "args", "n", "every")


class _Plan:
    __slots__ = ("params", "identity", "dtypes", "keys", "sizes", "numels", "buckets", "device", "streams", "captured", "covered", "state",
                 "memory", "keep")


class AdamW:
    """AdamW over any number of tensors (a list, or groups: dicts with `params` and optionally `name`, `lr`, `betas`, `eps`,
    `weight_decay`), updated in one launch per 352 tensors and 14 groups of a type:

        m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2;  p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    with g = grad * `grad_scale`.  `state_bits=8` keeps both moments in 8 bits, blocks of 256 elements sharing a power-of-two scale
    (2.01 instead of 8 bytes per parameter), rounded stochastically from `seed`, the step and the element's place: the same run
    gives the same bits.  `master_weights=True` keeps fp32 copies of 16-bit parameters and updates those; without, the update is
    rounded into the 16-bit parameter.  `lr` may be a float32 device scalar (a captured step reads it at replay).

    `state[key]`: `step` (int32 on the device), `exp_avg`, `exp_avg_sq` (float32, or uint8 codes with `exp_avg_scale` /
    `exp_avg_sq_scale`), `master`; key = the group's name if the group has one tensor, else "<name or number>.<i>".  A 16-bit
    parameter that is changed from outside between steps does not change its master: delete `state[key]["master"]`, and the
    next step takes it from the parameter again.
    Parameters must be contiguous; gradients of another layout are copied.  Tensors without a gradient are skipped, and so are
    their counters, as in torch.  A tensor of the state, or of the parameters, may be replaced, also its storage under it (`.data = `,
    `set_`): the next step sees it and looks at its tensors anew, which costs host work and one wait for the stream and cannot be
    captured.  Tensors that a step would write must not share memory.  `seed` and the groups' rates may be changed at any time;
    `state_bits` and `master_weights` are fixed.
    Memory: plan and state belong to the optimizer, which must live as long as graphs of its steps are replayed; a captured step writes
    the storages it was captured with (and holds the rates of its groups as they were, but for those given as device scalars).  One
    optimizer's steps are one sequence: two that run at the same time on two streams, or two of its captured graphs replayed so,
    race on the parameters."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master_weights=False, seed=0):
        params = list(params)
        if not params:
            raise ValueError("AdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits = {state_bits}: 8 or 32")
        self.defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
        groups = params if isinstance(params[0], dict) else [dict(params=params)]
        self.param_groups = [self._filled(g) for g in groups]
        self._state_bits, self._master_weights, self.seed = int(state_bits), bool(master_weights), int(seed) & 0xFFFFFFFF
        self.grad_scale = 1.0
        self._plan, self._captured, self._rates = None, [], None
        self._state_dict = _Watched(self)
        self._check_groups()

    def _check_groups(self):
        for k, g in enumerate(self.param_groups):
            self._hyper(k, g)
        seen = set()
        for p in self._tensors():
            if not isinstance(p, torch.Tensor):
                raise TypeError(f"AdamW: a {type(p).__name__} among the parameters")
            if id(p) in seen:
                raise ValueError("AdamW: a parameter appears twice")
            seen.add(id(p))

    def add_param_group(self, group):
        """One more group (a dict with `params`), with this optimizer's defaults for what it does not say."""
        self.param_groups.append(self._filled(group))
        try:
            self._check_groups()
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def _filled(self, g):
        if not isinstance(g, dict) or "params" not in g:
            raise TypeError("AdamW: groups are dictionaries with `params`")
        ps = g["params"]
        g["params"] = [ps] if isinstance(ps, torch.Tensor) else list(ps)
        for k, v in self.defaults.items():
            g.setdefault(k, v)
        return g

    def __getstate__(self):          # (copies and pickles: plans hold addresses and are made anew)
        return dict(self.__dict__, _plan=None, _captured=[], _rates=None, _state_dict={k: dict(v) for k, v in self.state.items()})

    def __setstate__(self, d):
        self.__dict__.update(d)
        self.state = d["_state_dict"]

    # ---- what is trained ---------------------------------------------------------------------------------------------
    # (what the state is held in: fixed, as the tensors of `state` are of that kind)
    state_bits = property(lambda self: self._state_bits)
    master_weights = property(lambda self: self._master_weights)

    @property
    def state(self):
        return self._state_dict

    @state.setter
    def state(self, new):
        self._plan = None
        self._state_dict = _Watched(self, {k: _Watched(self, v) for k, v in new.items()})

    def _tensors(self):
        return [p for g in self.param_groups for p in g["params"]]

    def _keys(self):
        out = []
        for i, g in enumerate(self.param_groups):
            name, n = str(g.get("name", i)), len(g["params"])
            out += [name] if n == 1 else [f"{name}.{j}" for j in range(n)]
        if len(set(out)) != len(out):
            raise ValueError(f"AdamW: group names are not unique: {sorted(k for k in set(out) if out.count(k) > 1)}")
        return out

    @staticmethod
    def _hyper(k, g):
        lr, (b1, b2), eps, wd = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        dev = None
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError(f"AdamW: group {k}: a tensor `lr` must be one float32 element on the device")
            dev, lr = lr.data_ptr(), 0.0
        if not (lr >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and (eps == 0.0 or eps >= 2.0 ** -126) and wd >= 0.0):
            raise ValueError(f"AdamW: group {k}: lr {lr}, betas {(b1, b2)}, eps {eps}, weight_decay {wd} out of range")
        return _lib.VcrOptimGroup(float(lr), float(b1), float(b2), float(eps), float(wd), dev)

    def _fresh(self, p):
        dev, n = p.device, p.numel()
        st = dict(step=torch.zeros((), dtype=torch.int32, device=dev))
        if self.state_bits == 32:
            st.update(exp_avg=torch.zeros(p.shape, device=dev), exp_avg_sq=torch.zeros(p.shape, device=dev))
        else:
            nb = -(-n // BLOCK)
            st.update({k: torch.zeros(p.shape, dtype=torch.uint8, device=dev) for k in ("exp_avg", "exp_avg_sq")})
            st.update({k: torch.ones(nb, dtype=torch.uint8, device=dev) for k in ("exp_avg_scale", "exp_avg_sq_scale")})
        if self._has_master(p):
            st["master"] = p.detach().float().contiguous()
        return _Watched(self, st)

    def _has_master(self, p):
        return self.master_weights and p.dtype != torch.float32

    def _check_state(self, key, p, st):
        """-> names of the tensors of the parameter's state that a step reads and writes."""
        n, nb = p.numel(), -(-p.numel() // BLOCK)
        want = {"step": (torch.int32, 1)}
        kind = torch.float32 if self.state_bits == 32 else torch.uint8
        want.update(exp_avg=(kind, n), exp_avg_sq=(kind, n))
        if self.state_bits == 8:
            want.update(exp_avg_scale=(kind, nb), exp_avg_sq_scale=(kind, nb))
        if self._has_master(p):
            want["master"] = (torch.float32, n)
        for k, (dt, m) in want.items():
            t = st.get(k)
            if not isinstance(t, torch.Tensor) or t.dtype != dt or t.numel() != m or t.device != p.device or not t.is_contiguous():
                raise ValueError(f"AdamW: state[{key!r}][{k!r}] must be {m} contiguous elements of {dt} on {p.device}")
        return list(want)

    def _build(self, identity, need):
        """Plan of all parameters that have a state, and of those in `need`, which get one.  `identity`: the native lists' words."""
        lib = _lib.load()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the first step after its tensors changed cannot be captured; take one step before the capture")
        keys, groups_of = self._keys(), [i for i, g in enumerate(self.param_groups) for _ in g["params"]]
        plan = _Plan()
        plan.params = self._tensors()
        plan.dtypes, plan.device = _check_list(plan.params, "params")
        plan.keys, plan.captured = keys, False
        plan.sizes, plan.numels, plan.identity = [len(g["params"]) for g in self.param_groups], [p.numel() for p in plan.params], identity
        if len(set(map(id, plan.params))) != len(plan.params):
            raise ValueError("AdamW: a parameter appears twice")
        self._check_dense(plan.params)
        by, plan.state, plan.keep, names, stepped, fresh = {}, [], [], [], [], []
        for i, (p, key) in enumerate(zip(plan.params, keys)):
            if key not in self.state:
                if i not in need:
                    continue
                dict.__setitem__(self.state, key, self._fresh(p))
                fresh.append(key)
            st = self.state[key]
            if type(st) is not _Watched:
                st = _Watched(self, st)
                dict.__setitem__(self.state, key, st)
            if self._has_master(p) and "master" not in st:
                dict.__setitem__(st, "master", p.detach().float().contiguous())
            held = self._check_state(key, p, st)
            plan.state += [st[k] for k in held]
            names += [f"state[{key!r}][{k!r}]" for k in held]
            stepped.append(i)
            by.setdefault(_TYPES[p.dtype], []).append(i)
        plan.buckets, plan.covered = [], sum(map(len, by.values()))
        twice = _native().sharing(plan.state, [plan.params[i] for i in stepped])
        if twice:
            names += [f"parameter {keys[i]!r}" for i in stepped]
            for key in fresh:
                dict.__delitem__(self.state, key)
            raise ValueError(f"AdamW: {' and '.join(names[i] for i in twice)} share memory: one launch would write it twice, in no order")
        plan.memory = _native().memory(plan.state)
        for kind, at in by.items():
            b = _Bucket()
            b.type, b.at, b.n, b.every = kind, at, len(at), len(at) == len(plan.params)
            b.numels, b.kinds = array("q", [plan.numels[i] for i in at]), array("i", [kind]) * b.n
            b.group_of = array("i", [groups_of[i] for i in at])
            rec = (_lib.VcrOptimTensor * b.n)()
            for r, i in zip(rec, at):
                p, st = plan.params[i], self.state[keys[i]]
                ptr = lambda k: st[k].data_ptr() if k in st else None  # noqa: E731
                r.p, r.master, r.numel, r.group, r.index = p.data_ptr(), ptr("master") if self._has_master(p) else None, p.numel(), groups_of[i], i
                r.m, r.v, r.step = ptr("exp_avg"), ptr("exp_avg_sq"), ptr("step")
                if self.state_bits == 8 and p.numel():
                    r.m_scale, r.v_scale = ptr("exp_avg_scale"), ptr("exp_avg_sq_scale")
            size = lib.vcr_optim_plan_bytes(b.n, _address(b.numels))
            host = torch.empty(size, dtype=torch.uint8)
            _lib.check(lib.vcr_optim_plan(b.n, rec, host.data_ptr(), size))
            b.plan = host.to(plan.device)
            b.args = _lib.VcrAdamWStep(ntensors=b.n, param_type=kind, state_bits=self.state_bits,
                                       masters=int(self.master_weights and kind != 0), plan=b.plan.data_ptr(),
                                       numel=_address(b.numels), group_of=_address(b.group_of))
            plan.buckets.append(b)
        torch.cuda.current_stream(plan.device).synchronize()          # (the upload is finished whatever stream the steps use)
        plan.streams = set()                     # (those that use it: none yet, the state may come from another than this one)
        self._plan = plan
        return plan

    def _current(self, params, words, flags):
        """The plan, rebuilt where a parameter or a state entry is another tensor than it holds or has other memory, or where one that is
        to be stepped (has a gradient and a flag) is not in it."""
        plan, identity = self._plan, words[8 * len(params):]
        fits = (plan is not None and plan.identity == identity and [len(g["params"]) for g in self.param_groups] == plan.sizes
                and _native().in_place(plan.state, plan.memory))
        if not fits or plan.covered < len(params):
            need = {i for i, p in enumerate(params) if p.grad is not None and (flags is None or flags[i])}
            if not fits or not need <= {i for b in plan.buckets for i in b.at}:
                plan = self._build(identity, need)
        stream = _stream(plan.device.index)
        if stream not in plan.streams:          # (what is freed later is not given away before this stream is done with it)
            plan.streams.add(stream)
            for t in plan.state + [b.plan for b in plan.buckets]:
                t.record_stream(torch.cuda.current_stream(plan.device))
        if torch.cuda.is_current_stream_capturing():        # the graph holds these addresses
            plan.keep += [g["lr"] for g in self.param_groups if isinstance(g["lr"], torch.Tensor)]
            if not plan.captured:                           # (aliases: they hold the memory whatever becomes of the tensors)
                plan.captured = True
                plan.keep += [t.detach() for t in plan.state + plan.params]
                self._captured.append(plan)
        return plan, stream

    def _group_table(self, device):
        """The groups' rates as the library takes them, formed anew only where one has changed."""
        key = [(float(lr) if not isinstance(lr, torch.Tensor) else (lr.data_ptr(), lr.dtype, lr.numel(), lr.device), *g["betas"], g["eps"],
                g["weight_decay"]) for g in self.param_groups for lr in (g["lr"],)]
        if self._rates is None or self._rates[0] != key:
            for k, g in enumerate(self.param_groups):
                if isinstance(g["lr"], torch.Tensor) and g["lr"].device != device:
                    raise ValueError(f"AdamW: group {k}: `lr` is on {g['lr'].device}, the parameters are on {device}")
            self._rates = key, (_lib.VcrOptimGroup * len(key))(*[self._hyper(k, g) for k, g in enumerate(self.param_groups)])
        return self._rates[1]

    # ---- the step -----------------------------------------------------------------------------------------------------
    def step(self, only=None, max_norm=None):
        """One update of every parameter that has a gradient (`only`: of the groups with these names; their gradients are released
        afterwards, as in `FusedAdam.step`).  `max_norm`: the gradients count with the factor min(1, max_norm / (norm + 1e-6)), norm the
        2-norm of all gradients of this step times `grad_scale`; -> the norm (0-dim float32; nothing waits for it), and if that is not
        finite in float32 the whole step is skipped on the device: parameters, moments and counters stay.  Infinity as `max_norm`
        measures and guards, and never clips.  Without `max_norm`: -> None."""
        if max_norm is not None:
            max_norm = _positive(max_norm, "max_norm")
        params, flags = self._tensors(), None
        if only is not None:
            only = {only} if isinstance(only, str) else set(only)
            flags = bytes(g.get("name") in only for g in self.param_groups for _ in g["params"])
        found = _native().gradients(params, flags)
        if found is None:
            if all(p.grad is None or (flags and not f) for p, f in zip(params, flags or params)):
                return None
            found = self._looked_at(params, flags)
        _, live, words, at, *_holds = found
        if not live:
            return None
        plan, stream = self._current(params, words, flags)
        norm = _on(plan.device, self._launch, plan, words, at, live, max_norm, stream)
        _native().changed(params, words)
        if only is not None:
            for p, f in zip(params, flags):
                if f:
                    p.grad = None
        return norm

    def _looked_at(self, params, flags):
        """What `gradients` of the native lists gives, for lists that are not ordinary: dense copies of gradients, or what is wrong."""
        dtypes, dev = _check_list(params, "params")
        self._check_dense(params)
        live = [i for i, p in enumerate(params) if p.grad is not None and (flags is None or flags[i])]
        work = _dense([params[i].grad for i in live], "AdamW: gradients")
        grads = array("Q", bytes(8 * len(params)))
        for i, g in zip(live, work):
            if g.dtype is not dtypes[i] or g.numel() != params[i].numel() or g.device != dev:
                raise ValueError(f"AdamW: the gradient of {self._keys()[i]!r} has type {g.dtype} and {g.numel()} elements on {g.device}, "
                                 f"the parameter {dtypes[i]} and {params[i].numel()} on {dev}")
            grads[i] = g.data_ptr() if g.numel() else 1
            if not grads[i]:
                raise ValueError(f"AdamW: the gradient of {self._keys()[i]!r} has no memory")
        words = b"".join(a.tobytes() for a in (grads, array("Q", map(id, params)), array("Q", [p.data_ptr() for p in params]),
                                               array("q", [p.numel() for p in params]), array("i", [_TYPES[d] for d in dtypes])))
        return dev.index, len(live), words, C.cast(words, C.c_void_p).value, work

    def _check_dense(self, params):
        for key, p in zip(self._keys(), params):
            if not p.is_contiguous() or p.is_neg():
                raise ValueError(f"AdamW: parameter {key!r} is not contiguous")

    def _launch(self, plan, words, at, live, max_norm, stream):
        groups, lib, norm, clip, n = self._group_table(plan.device), _lib.load(), None, None, len(plan.params)
        grads = None if live == n and len(plan.buckets) == 1 else memoryview(words)[:8 * n].cast("Q")
        if max_norm is not None:
            norm = torch.empty((), device=plan.device)
            if live == n:
                args = n, at, at + 24 * n, at + 32 * n
            else:
                some = [i for i in range(n) if grads[i]]
                lists = (array("Q", [grads[i] for i in some]), array("q", [plan.numels[i] for i in some]),
                         array("i", [_TYPES[plan.dtypes[i]] for i in some]))
                args = len(some), *map(_address, lists)
            clip = _norm(args, norm, stream, True, float(self.grad_scale), max_norm, True)
        for b in plan.buckets:
            mine = None if b.every else array("Q", [grads[i] for i in b.at])
            a = b.args
            a.grads, a.groups, a.ngroups, a.grad_scale = at if b.every else _address(mine), groups, len(groups), float(self.grad_scale)
            a.seed = self.seed & 0xFFFFFFFF
            a.clip = None if clip is None else clip.data_ptr()
            _lib.check(lib.vcr_adamw_step(C.byref(a), stream))
        return norm

    def zero_grad(self, set_to_none=True):
        for p in self._tensors():
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    # ---- moments as values ---------------------------------------------------------------------------------------------
    def moments(self, exp_avgs=None, exp_avg_sqs=None, dtype=torch.float32):
        """The moments as values, whatever they are held in: two lists, one tensor for each parameter in the groups' order.  Given
        lists are written to (contiguous, all of one type, sharing no memory) instead of new tensors of `dtype`; a parameter that has not
        been stepped yet has zeros.  8-bit moments are exact in bfloat16."""
        params, native = self._tensors(), _native()
        n, none = len(params), bytes(len(params))
        for given in (exp_avgs, exp_avg_sqs):
            if given is not None:
                dtype = given[0].dtype if len(given) else dtype
                if len(given) != n:
                    raise ValueError(f"moments: {len(given)} tensors for {n} parameters")
        outs = [[torch.empty(p.shape, dtype=dtype, device=p.device) for p in params] if given is None else given
                for given in (exp_avgs, exp_avg_sqs)]
        lists = [o if type(o) is list else list(o) for o in outs]
        a, c = found = [native.words(o) for o in lists]          # device, words, their address
        kind = None if None in found else a[1][16 * n:16 * n + 4]
        if kind is None or not a[1][16 * n:] == c[1][16 * n:] == kind * n:
            kinds = {t.dtype for o in outs for t in o}
            if len(kinds) != 1 or not kinds <= _TYPES.keys():
                raise ValueError(f"moments: the outputs must be of one type among float32, bfloat16, float16: {kinds}")
        plan, stream = self._current(params, (native.gradients(params, none) or self._looked_at(params, none))[2], none)
        sizes = plan.identity[16 * n:24 * n]
        if None in found or not (a[0] == c[0] == plan.device.index and a[1][8 * n:16 * n] == c[1][8 * n:16 * n] == sizes):
            raise ValueError("moments: an output has another size or device than its parameter, or is not contiguous")
        twice = None if exp_avgs is exp_avg_sqs is None else native.sharing(*lists)
        if twice:
            raise ValueError(f"moments: outputs {twice[0]} and {twice[1]} (counted through both lists) share memory")
        if plan.covered < len(params):
            held = {i for b in plan.buckets for i in b.at}
            for i in range(len(params)):
                if i not in held:
                    outs[0][i].detach().zero_()
                    outs[1][i].detach().zero_()
        if self.state_bits == 32:
            for b in plan.buckets:
                for i in b.at:
                    for o, k in zip(outs, ("exp_avg", "exp_avg_sq")):
                        o[i].detach().copy_(self.state[plan.keys[i]][k].view(o[i].shape))
        else:
            kind = int.from_bytes(kind, sys.byteorder)
            for b in plan.buckets:
                some = None if b.every else [array("Q", [o[i].data_ptr() for i in b.at]) for o in outs]
                m, v = (a[2], c[2]) if b.every else map(_address, some)
                _lib.check(_on(plan.device, _lib.load().vcr_moments8_decode, b.n, b.plan.data_ptr(), _address(b.numels), m, v, kind, stream))
            for given, o in zip((exp_avgs, exp_avg_sqs), lists):
                if given is not None:
                    native.changed(o, None)
        return outs

    @torch.no_grad()
    def moments_of(self, key):
        """The two moments of one parameter, by the state's key: the float32 tensors themselves, or what the 8-bit codes stand for."""
        st = self.state[key]
        if self.state_bits == 32:
            return st["exp_avg"], st["exp_avg_sq"]
        return tuple(decode8(st))

    @torch.no_grad()
    def set_moments(self, key, exp_avg, exp_avg_sq, step=None):
        """Gives the parameter of `key` these moments (float32 values of its shape; 8 bits: rounded to the nearest code)."""
        keys = self._keys()
        if key not in keys:
            raise KeyError(f"AdamW: no parameter {key!r}")
        p = self._tensors()[keys.index(key)]
        for t in (exp_avg, exp_avg_sq):
            if t.numel() != p.numel():
                raise ValueError(f"set_moments: {t.numel()} values for the {p.numel()} elements of {key!r}")
        old = self.state.get(key)
        st = self._fresh(p)
        if old is not None:
            st["step"] = old["step"]
            if "master" in old and old["master"].numel() == p.numel():
                st["master"] = old["master"]
        if step is not None:
            st["step"].fill_(int(step))
        given = [t.detach().reshape(p.shape) for t in (exp_avg, exp_avg_sq)]
        if self.state_bits == 32:                            # (copied: the caller's tensors stay the caller's, also one given twice)
            for k, t in zip(("exp_avg", "exp_avg_sq"), given):
                st[k].copy_(t)
        elif p.numel():
            encode8(*(t.to(device=p.device, dtype=torch.float32).contiguous() for t in given), st)
        self.state[key] = st

    # ---- checkpoints -----------------------------------------------------------------------------------------------------
    def state_dict(self):
        """torch.optim.AdamW's layout (state by running index, `step` a float32 scalar).  8-bit moments are stored as they are held
        (uint8 codes and scales); `moments()` gives the values another optimizer could load."""
        template = torch.optim.AdamW([torch.zeros(1)]).param_groups[0]
        state, groups, idx = {}, [], 0
        held = [(i, self.state[key]) for i, key in enumerate(self._keys()) if key in self.state]
        steps = torch.stack([st["step"].reshape(()) for _, st in held]).tolist() if held else []          # (one wait for all)
        for (i, st), t in zip(held, steps):
            state[i] = {k: torch.tensor(float(t)) if k == "step" else v for k, v in st.items()}
        for g in self.param_groups:
            wg = {k: v for k, v in template.items() if k != "params"}
            wg.update({k: v for k, v in g.items() if k != "params"})
            wg["params"] = list(range(idx, idx + len(g["params"])))
            idx += len(g["params"])
            groups.append(wg)
        return dict(state=state, param_groups=groups)

    @torch.no_grad()
    def load_state_dict(self, sd):
        """Takes what `state_dict()` gave -- or torch.optim.AdamW's: float moments are rounded into the 8-bit form where this optimizer
        has that, and 8-bit ones expanded where it has not.  Tensors that already have this optimizer's type, layout and device are
        kept, not copied, as torch does; a rate that is a tensor is copied.  Groups are matched in order, shapes must be the parameters'.
        Files of torch's `amsgrad` and `maximize` variants are refused."""
        if len(sd["param_groups"]) != len(self.param_groups):
            raise ValueError(f"AdamW: {len(sd['param_groups'])} groups saved, {len(self.param_groups)} here")
        order = []
        for k, (wg, g) in enumerate(zip(sd["param_groups"], self.param_groups)):
            if len(wg["params"]) != len(g["params"]):
                raise ValueError(f"AdamW: group {k}: {len(wg['params'])} tensors saved, {len(g['params'])} here")
            self._check_saved(wg)
            order += list(wg["params"])
        new = {}
        held = [(key, p, sd["state"][i]) for i, key, p in zip(order, self._keys(), self._tensors()) if i in sd["state"]]
        if held:
            steps = torch.tensor([int(round(float(st["step"]))) for _, _, st in held], dtype=torch.int32).to(held[0][1].device).unbind()
            for (key, p, st), t in zip(held, steps):
                new[key] = self._converted(key, p, st, t)
        for wg, g in zip(sd["param_groups"], self.param_groups):
            for k in ("lr", "eps", "weight_decay"):
                if k in wg:
                    g[k] = wg[k]
            if "lr" in wg and isinstance(g["lr"], torch.Tensor):            # (the optimizer's own, on its device, wherever the file was read to)
                dev = g["params"][0].device if g["params"] else g["lr"].device
                g["lr"] = g["lr"].detach().to(device=dev, dtype=torch.float32, copy=True)
            if "betas" in wg:
                g["betas"] = tuple(wg["betas"])
        self.state = new

    @staticmethod
    def _check_saved(wg):
        for k in ("amsgrad", "maximize"):
            if wg.get(k):
                raise ValueError(f"AdamW: the checkpoint's optimizer ran with {k}=True, which this one does not do")

    def _converted(self, key, p, st, step):
        dev, n, nb = p.device, p.numel(), -(-p.numel() // BLOCK)
        for k in ("exp_avg", "exp_avg_sq"):              # (the shape: moments in another order fit by their number alone)
            if tuple(st[k].shape) != tuple(p.shape):
                raise ValueError(f"optimizer state of {key!r} has shape {tuple(st[k].shape)}, parameter {tuple(p.shape)}")
        out = dict(step=step)
        as_held = lambda t, dt: t.detach().to(device=dev, dtype=dt).contiguous()  # noqa: E731
        codes = st["exp_avg"].dtype == torch.uint8
        if codes:
            raw = {k: as_held(st[k], torch.uint8) for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
            if any(raw[k].numel() != nb for k in ("exp_avg_scale", "exp_avg_sq_scale")):
                raise ValueError(f"optimizer state of {key!r}: {nb} block scales expected")
            out.update(raw)
            if self.state_bits == 32:
                out.update(zip(("exp_avg", "exp_avg_sq"), decode8(raw)))
                del out["exp_avg_scale"], out["exp_avg_sq_scale"]
        else:
            m, v = as_held(st["exp_avg"], torch.float32), as_held(st["exp_avg_sq"], torch.float32)
            if self.state_bits == 32:
                out.update(exp_avg=m, exp_avg_sq=v)
            else:
                out.update({k: torch.zeros(p.shape, dtype=torch.uint8, device=dev) for k in ("exp_avg", "exp_avg_sq")})
                out.update({k: torch.ones(nb, dtype=torch.uint8, device=dev) for k in ("exp_avg_scale", "exp_avg_sq_scale")})
                encode8(m, v, out)
        if self._has_master(p):
            if "master" in st and tuple(st["master"].shape) != tuple(p.shape):
                raise ValueError(f"optimizer state of {key!r}: the master has shape {tuple(st['master'].shape)}, parameter {tuple(p.shape)}")
            out["master"] = as_held(st["master"], torch.float32) if "master" in st else p.detach().float().contiguous()
        return out


def _check_codes(st):
    """-> elements and device of the 8-bit moments in `st`, whose four tensors must fit each other."""
    n, dev = st["exp_avg"].numel(), st["exp_avg"].device
    nb = -(-n // BLOCK)
    for k, m in (("exp_avg", n), ("exp_avg_sq", n), ("exp_avg_scale", nb), ("exp_avg_sq_scale", nb)):
        t = st[k]
        if t.dtype != torch.uint8 or t.numel() != m or t.device != dev or not t.is_contiguous():
            raise ValueError(f"8-bit moments: {k!r} must be {m} contiguous elements of torch.uint8 on {dev}")
    if dev.type != "cuda":
        raise ValueError("8-bit moments need a HIP device")
    return n, dev


def _single(st, n, dev):
    """A plan of one tensor's 8-bit moments, for the code <-> value kernels."""
    lib = _lib.load()
    rec = (_lib.VcrOptimTensor * 1)()
    rec[0].p = rec[0].m = st["exp_avg"].data_ptr()
    rec[0].v, rec[0].m_scale, rec[0].v_scale = (st[k].data_ptr() for k in ("exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"))
    rec[0].step = st["exp_avg"].data_ptr()               # (not used by these kernels, but not optional)
    rec[0].numel = n
    ns = array("q", [n])
    size = lib.vcr_optim_plan_bytes(1, _address(ns))
    host = torch.empty(size, dtype=torch.uint8)
    _lib.check(lib.vcr_optim_plan(1, rec, host.data_ptr(), size))
    return host.to(dev), ns


def encode8(exp_avg, exp_avg_sq, st):
    """float32 moments into the uint8 tensors `exp_avg`, `exp_avg_sq`, `exp_avg_scale`, `exp_avg_sq_scale` of `st`, to the nearest."""
    for k, t in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
        if t.dtype != torch.float32 or t.numel() != st["exp_avg"].numel() or t.device != st["exp_avg"].device or not t.is_contiguous():
            raise ValueError(f"encode8: the values of {k!r} must be {st['exp_avg'].numel()} contiguous elements of torch.float32 on "
                             f"{st['exp_avg'].device}")
    n, dev = _check_codes(st)
    if n:
        plan, ns = _single(st, n, dev)
        m, v = array("Q", [exp_avg.data_ptr()]), array("Q", [exp_avg_sq.data_ptr()])
        _lib.check(_on(dev, _lib.load().vcr_moments8_encode, 1, plan.data_ptr(), _address(ns), _address(m), _address(v),
                       _lib.stream_of(st["exp_avg"])))


def decode8(st):
    """-> the float32 values of the 8-bit moments in `st`, of their shape."""
    n, dev = _check_codes(st)
    outs = [torch.empty(st["exp_avg"].shape, device=dev) for _ in range(2)]
    if n:
        plan, ns = _single(st, n, dev)
        m, v = (array("Q", [o.data_ptr()]) for o in outs)
        _lib.check(_on(dev, _lib.load().vcr_moments8_decode, 1, plan.data_ptr(), _address(ns), _address(m), _address(v), 0,
                       _lib.stream_of(st["exp_avg"])))
    return outs


def rows8(states, index):
    """8-bit moments with their rows (along the first dimension) in another order: for each of `states` (dicts as `decode8`'s, all of the
    same number of rows) new tensors whose row r is row index[r] of the old ones; zeros where index[r] is no row (-1).  By code: blocks
    are formed anew, to the nearest, and nothing is expanded on the way."""
    if index.dtype != torch.int32 or index.dim() != 1 or not index.is_contiguous():
        raise ValueError("rows8: `index` must be a contiguous vector of int32")
    shapes = [st["exp_avg"].shape for st in states]
    if any(len(s) == 0 or s[0] != shapes[0][0] or st["exp_avg_sq"].shape != s for st, s in zip(states, shapes)):
        raise ValueError("rows8: moments of one number of rows, both of a parameter's shape, are needed")
    arr, new = (_lib.VcrRows8 * len(states))(), []
    for a, st, shape in zip(arr, states, shapes):
        _check_codes(st)
        if st["exp_avg"].device != index.device:
            raise ValueError(f"rows8: moments on {st['exp_avg'].device}, `index` on {index.device}")
        out = {k: torch.empty((index.numel(), *shape[1:]), dtype=torch.uint8, device=index.device) for k in ("exp_avg", "exp_avg_sq")}
        blocks = -(-out["exp_avg"].numel() // BLOCK)
        out.update({k: torch.empty(blocks, dtype=torch.uint8, device=index.device) for k in ("exp_avg_scale", "exp_avg_sq_scale")})
        a.width = shape[1:].numel()
        for k, i, o in (("exp_avg", "m", "m_out"), ("exp_avg_sq", "v", "v_out"), ("exp_avg_scale", "m_scale", "m_scale_out"),
                        ("exp_avg_sq_scale", "v_scale", "v_scale_out")):
            setattr(a, i, st[k].data_ptr())
            setattr(a, o, out[k].data_ptr())
        new.append(out)
    live = [a for a in arr if a.width]                       # (rows without elements: nothing to move)
    if live:
        _lib.check(_on(index.device, _lib.load().vcr_moments8_rows, len(live), (_lib.VcrRows8 * len(live))(*live), shapes[0][0],
                       index.numel(), index.data_ptr(), _stream(index.device.index)))
    return new
