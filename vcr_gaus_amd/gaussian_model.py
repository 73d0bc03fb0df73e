"""GaussianModel: same operator surface as the reference's `scene/gaussian_model.py`
(getters, Adam parameter groups, densify / prune surgery, densification statistics), with the
per-step arithmetic routed to HIP kernels:

  * activations + shortest-axis normal + camera orientation: one fused kernel each way
    (`fused_activate`, replaces `scene/gaussian_model.py:125-192` + `gaussian_renderer/__init__.py:95-101`)
  * Adam over all parameter groups: one launch (`FusedAdam`, replaces `torch.optim.Adam` at `:258`); on request AdamW instead
    (`GaussianAdamW`: decoupled weight decay, clipping, moments in 8 bits)
  * densification statistics: one kernel (`add_densification_stats`, `:669-671` + `trainer.py:345`)

  * densify / prune row surgery: parameters, both Adam moments and the statistics of ALL groups re-packed by one
    plan + one move launch (`_move_rows`, replaces `_prune_optimizer` / `cat_tensors_to_optimizer`, `:425-531`)

The selection rules (gradient threshold, clone / deterministic two-way split, prune masks) are the reference's
(`scene/gaussian_model.py:579-667`) as a handful of small torch ops on the device.
"""
import ctypes as C

import numpy as np
import torch

from . import _lib
from .general_utils import build_rotation, get_expon_lr_func, inverse_sigmoid
from .optim import AdamW, rows8

GROUPS = ["xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation", "obj_dc"]


class GeometrySink:
    """Everything ONE training iteration hands from node to node outside autograd's tensors -- one object per iteration,
    owned by the trainer (`model._geom_sink` while the step runs); nothing process-global.
      * `defer_scale_grad` / `scale_grad`: the l1_scale regulariser of the fused loss node reaches `_scaling` on a second path;
        instead of a second incoming gradient on that leaf (an add kernel of the engine) the loss node leaves it here and the
        backward of the fused activation -- same graph, runs later -- adds it inside its own kernel;
      * `armed` + `grads` / `saved` / `scale_reg`: the fused static tail.  With an ARMED sink the activation backward does not
        launch its kernel but leaves the upstream gradients (w.r.t. activated scales / rotations / opacities / camera normals)
        and what it saved, and the loss node leaves the FACTORS of the l1_scale gradient; `FusedAdam.geometry_step` consumes both;
      * `tail` / `done`: the same tail INSIDE the rasterizer's backward (`vcr_rasterize_backward_tail`): `tail()` -> the
        argument block + commit of `FusedAdam.prepare_geometry_step(in_registers=True)`; the rasterizer node (which holds this
        sink through its `RasterOptions`) calls it, sets `done`, and returns no gradient for means / scales / rotations /
        opacities / normals, so the activation backward has nothing left to do.  NOT atomic with the rest of the step: Adam on
        xyz / scaling / rotation / opacity is applied in the middle of `loss.backward()`; if anything raises later in the same
        backward or in the gradient exchange, the geometry has been stepped and the SH coefficients have not -- `started` is
        set before the launch and the trainer then reports `last_tail = "raster-partial"`: such a step must not be retried;
      * `sums`: the trainer's cache of the loss node's fp64 reduction buffer, {device: [buffer, in use]} (re-zeroed by the
        finalize kernel, so it can be re-used from step to step instead of being allocated and cleared)."""
    __slots__ = ("armed", "grads", "saved", "scale_reg", "defer_scale_grad", "scale_grad", "sums", "tail", "done", "want_normal",
                 "started", "exchange")

    def __init__(self, armed=True, defer_scale_grad=False, sums=None, tail=None):
        self.armed, self.grads, self.saved, self.scale_reg = armed, None, None, None
        self.defer_scale_grad, self.scale_grad, self.sums = defer_scale_grad, None, sums
        self.tail, self.done, self.want_normal = tail, False, None
        self.exchange = False         # data parallel: the rasterizer's backward writes dL/dnormals in world space (see Trainer)
        self.started = False          # set right before the tail's launch inside the rasterizer's backward (see `Trainer.last_tail`)


class _FusedActivate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scaling, rotation, opacity, xyz, campos, R_w2c, want_normal, sink=None, pre=None):
        lib = _lib.load()
        N = xyz.shape[0]
        dev = xyz.device
        sr, rr, orr = scaling.detach().contiguous(), rotation.detach().contiguous(), opacity.detach().contiguous()
        Rw = R_w2c.detach().contiguous().float()
        if pre is not None:           # the previous iteration's static tail has already evaluated this (ActivationCache)
            scales, rots, opac, nrm, aux = pre
        else:
            scales = torch.empty(N, 3, device=dev)
            rots = torch.empty(N, 4, device=dev)
            opac = torch.empty(N, 1, device=dev)
            nrm = torch.empty(N, 3, device=dev) if want_normal else None
            aux = torch.empty(N, dtype=torch.uint8, device=dev)
            cp = campos.detach().contiguous().float()
            _lib.check(lib.vcr_activate_forward(N, sr.data_ptr(), rr.data_ptr(), orr.data_ptr(), xyz.detach().contiguous().data_ptr(),
                                                cp.data_ptr(), Rw.data_ptr(), scales.data_ptr(), rots.data_ptr(), opac.data_ptr(),
                                                nrm.data_ptr() if want_normal else None, aux.data_ptr(), _lib.stream_of(xyz)))
        ctx.save_for_backward(sr, rr, orr, Rw, aux)
        ctx.set_materialize_grads(False)
        ctx.want_normal = want_normal
        ctx.sink = sink
        if sink is not None and sink.armed:
            sink.saved = (sr, rr, orr, Rw, aux)          # (the tail may run before this node's backward: inside the rasterizer's)
            sink.want_normal = want_normal
        if want_normal:
            return scales, rots, opac, nrm
        return scales, rots, opac

    @staticmethod
    def backward(ctx, d_scales, d_rots, d_opac, d_nrm=None):
        lib = _lib.load()
        if d_scales is None and d_rots is None and d_opac is None and d_nrm is None:
            return (None,) * 9                   # (e.g. the rasterizer's backward has applied the static tail itself)
        sr, rr, orr, Rw, aux = ctx.saved_tensors
        N = sr.shape[0]
        if ctx.sink is not None and ctx.sink.done:
            # the rasterizer's backward has already applied Adam to these parameters from ITS gradients; one that arrives here
            # now came by another path (a loss on the activated scales / opacities / normals that bypasses the rasterizer) and
            # would be dropped silently
            raise RuntimeError("fused geometry tail: a gradient reached the activated scales / rotations / opacities / normals "
                               "outside the rasterizer after the tail had run inside its backward; set "
                               "Trainer.fuse_geometry = False for such losses")
        keep = [None if t is None else t.contiguous().float() for t in (d_scales, d_rots, d_opac, d_nrm)]
        if ctx.sink is not None and ctx.sink.exchange and not (ctx.sink.armed and ctx.sink.grads is None):
            # (the rasterizer wrote dL/dnormals in the world-space form of the data-parallel exchange: only the one-kernel tail
            #  understands it)
            raise RuntimeError("fused geometry tail: the data-parallel exchange form was requested but the sink is not armed")
        if ctx.sink is not None and ctx.sink.armed and ctx.sink.grads is None:
            # fused static tail: `FusedAdam.geometry_step` applies this adjoint together with Adam in one pass
            ctx.sink.grads, ctx.sink.saved = keep, (sr, rr, orr, Rw, aux)
            return (None,) * 9
        ds, dr, do = torch.empty_like(sr), torch.empty_like(rr), torch.empty_like(orr)
        extra = None
        if ctx.sink is not None and ctx.sink.scale_grad is not None:          # l1_scale gradient of this iteration's loss node
            extra, ctx.sink.scale_grad = ctx.sink.scale_grad, None
            if tuple(extra.shape) != tuple(sr.shape):
                raise RuntimeError(f"pending l1_scale gradient has shape {tuple(extra.shape)}, the scaling parameter {tuple(sr.shape)}")
        _lib.check(lib.vcr_activate_backward(N, sr.data_ptr(), rr.data_ptr(), orr.data_ptr(), Rw.data_ptr(), aux.data_ptr(),
                                             *[None if t is None else t.data_ptr() for t in keep],
                                             None if extra is None else extra.data_ptr(),
                                             ds.data_ptr(), dr.data_ptr(), do.data_ptr(), _lib.stream_of(sr)))
        return ds, dr, do, None, None, None, None, None, None


class ActivationCache:
    """Activated scales / rotations / opacities (+ camera-space normals) that the static tail of the PREVIOUS iteration wrote
    for the camera of this one (`VcrGeometryStep.next_*`: the parameters are in registers there anyway).  One-shot: the next
    `fused_activate` on the model takes it if -- and only if -- it asks for the same camera tensors, the same `want_normal`
    and the raw parameters are the tensors (storage and version counter) the tail updated; anything else drops it."""
    __slots__ = ("campos", "R", "want_normal", "tensors", "stamp", "params")

    @staticmethod
    def stamp_of(pc):
        return tuple((t.data_ptr(), t._version, tuple(t.shape)) for t in (pc._scaling, pc._rotation, pc._opacity, pc._xyz))

    def __init__(self, pc, campos, R, want_normal, tensors):
        self.campos, self.R, self.want_normal, self.tensors = campos, R, want_normal, tensors
        self.stamp = self.stamp_of(pc)
        # the parameter OBJECTS the tail updated: the kernels write through raw pointers (the version counter stays 0), so a
        # rebuilt parameter that the caching allocator put at the same address would carry the same stamp
        self.params = (pc._scaling, pc._rotation, pc._opacity, pc._xyz)

    def matches(self, pc, campos, R, want_normal):
        return (campos is self.campos or campos.data_ptr() == self.campos.data_ptr()) and \
            (R is self.R or R.data_ptr() == self.R.data_ptr()) and bool(want_normal) == bool(self.want_normal) and \
            all(a is b for a, b in zip(self.params, (pc._scaling, pc._rotation, pc._opacity, pc._xyz))) and \
            self.stamp == self.stamp_of(pc)


def fused_activate(pc, camera_center, R_w2c, want_normal=True):
    """-> (scales[N,3], rotations[N,4], opacity[N,1], normals_cam[N,3]) from the raw parameters."""
    pre = None
    cache = getattr(pc, "_act_cache", None)
    if cache is not None:
        pc._act_cache = None
        if cache.matches(pc, camera_center, R_w2c, want_normal):
            pre = cache.tensors
    return _FusedActivate.apply(pc._scaling, pc._rotation, pc._opacity, pc._xyz, camera_center, R_w2c, want_normal,
                                getattr(pc, "_geom_sink", None), pre)


class FusedAdam:
    """`torch.optim.Adam(lr=0.0, eps=1e-15)` semantics with per-group learning rates
    (`scene/gaussian_model.py:247-258`), executed as ONE HIP launch over all groups.
    Keeps `param_groups` / `state` / `step()` / `zero_grad()` / `state_dict()` like the torch class."""

    def __init__(self, groups, eps=1e-15, betas=(0.9, 0.999)):
        self.param_groups = groups
        self.eps, self.betas = eps, betas
        self.state = {}          # name -> dict(step, exp_avg, exp_avg_sq)
        self.grad_scale = 1.0

    def _state(self, g):
        st = self.state.get(g["name"])
        if st is None:
            p = g["params"][0]
            st = dict(step=0, exp_avg=torch.zeros_like(p), exp_avg_sq=torch.zeros_like(p))
            self.state[g["name"]] = st
        return st

    @torch.no_grad()
    def step(self, only=None):
        """`only`: optional set of group names to update now (their gradients are released afterwards), used by the
        data-parallel trainer to run Adam on the SH groups while the other groups' all-reduce is still in flight."""
        lib = _lib.load()
        live = [g for g in self.param_groups if g["params"][0].grad is not None and g["params"][0].numel() > 0
                and (only is None or g["name"] in only)]
        if not live:
            return
        by_step = {}
        for g in live:
            st = self._state(g)
            st["step"] += 1
            by_step.setdefault(st["step"], []).append(g)
        for step, gs_all in by_step.items():
            for c0 in range(0, len(gs_all), 8):                      # vcr_adam_step takes at most 8 tensors per launch
                gs = gs_all[c0:c0 + 8]
                n = len(gs)
                P, G, M, V = ((C.c_void_p * n)() for _ in range(4))
                numel = (C.c_int64 * n)()
                lr = (C.c_float * n)()
                keep = []
                for k, g in enumerate(gs):
                    p = g["params"][0]
                    st = self.state[g["name"]]
                    grad = p.grad.contiguous()
                    keep.append(grad)
                    P[k], G[k], M[k], V[k] = p.data_ptr(), grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
                    numel[k], lr[k] = p.numel(), g["lr"]
                _lib.check(lib.vcr_adam_step(n, P, G, M, V, numel, lr, self.betas[0], self.betas[1], self.eps, step,
                                             float(self.grad_scale), _lib.stream_of(gs[0]["params"][0])))
        if only is not None:
            for g in live:
                g["params"][0].grad = None

    @torch.no_grad()
    def prepare_geometry_step(self, model, sink, grad2d=None, radii=None, in_registers=False, stats=False, next_cam=None,
                              normals_world=False):
        """-> (VcrGeometryStep, commit): the argument block of the static tail and the host bookkeeping to run once the launch
        has been accepted (Adam step counters, `_xyz.grad`).  `in_registers`: the form `vcr_rasterize_backward_tail` takes
        -- no upstream gradient arrays (they stay inside the projection-backward kernel), `stats` instead of `grad2d` /
        `radii`, and xyz always stepped.  `normals_world`: the data-parallel form -- `sink.grads` / `_xyz.grad` hold the
        all-reduced activated-space gradients, the normal gradient w.r.t. the world-space axis column
        (`RasterOptions.world_normals`); `self.grad_scale` (1 / world) is applied inside the kernel."""
        groups = {g["name"]: g for g in self.param_groups}
        sr, rr, orr, Rw, aux = sink.saved
        if in_registers:
            d_scales = d_rots = d_opac = d_nrm = None
        else:
            d_scales, d_rots, d_opac, d_nrm = sink.grads
        N = model._xyz.shape[0]
        for name, raw in (("scaling", sr), ("rotation", rr), ("opacity", orr)):
            if raw.data_ptr() != groups[name]["params"][0].data_ptr():
                raise RuntimeError(f"geometry_step: the backward saw another `{name}` tensor than the optimizer holds")
        gx = None if in_registers else model._xyz.grad
        step_xyz = in_registers or gx is not None
        st = {k: self._state(groups[k]) for k in ("xyz", "scaling", "rotation", "opacity")}
        # the counters are advanced only once the launch has been accepted: a failed call must not shift the bias correction
        nxt = {k: st[k]["step"] + (1 if (k != "xyz" or step_xyz) else 0) for k in st}
        ptr = lambda t: None if t is None else t.data_ptr()
        gxc = None if gx is None else gx.contiguous()
        sreg = sink.scale_reg
        want_stats = stats if in_registers else grad2d is not None
        a = _lib.VcrGeometryStep(
            N=N, normals_world=int(bool(normals_world)), grad_scale=float(self.grad_scale),
            step_xyz=nxt["xyz"] if step_xyz else 0, step_scaling=nxt["scaling"],
            step_rotation=nxt["rotation"], step_opacity=nxt["opacity"],
            xyz=model._xyz.data_ptr(), scaling=sr.data_ptr(), rotation=rr.data_ptr(), opacity=orr.data_ptr(),
            d_means3D=ptr(gxc), d_scales=ptr(d_scales), d_rots=ptr(d_rots), d_opac=ptr(d_opac), d_normals=ptr(d_nrm),
            aux=aux.data_ptr(), Rw2c=Rw.data_ptr(),
            scale_reg_gout=None if sreg is None else sreg["gout"], scale_reg_sums=None if sreg is None else sreg["sums"],
            trans=None if sreg is None else sreg["trans"].data_ptr(), scale=None if sreg is None else sreg["scale"].data_ptr(),
            m_xyz=st["xyz"]["exp_avg"].data_ptr(), v_xyz=st["xyz"]["exp_avg_sq"].data_ptr(),
            m_scaling=st["scaling"]["exp_avg"].data_ptr(), v_scaling=st["scaling"]["exp_avg_sq"].data_ptr(),
            m_rotation=st["rotation"]["exp_avg"].data_ptr(), v_rotation=st["rotation"]["exp_avg_sq"].data_ptr(),
            m_opacity=st["opacity"]["exp_avg"].data_ptr(), v_opacity=st["opacity"]["exp_avg_sq"].data_ptr(),
            lr_xyz=float(groups["xyz"]["lr"]), lr_scaling=float(groups["scaling"]["lr"]), lr_rotation=float(groups["rotation"]["lr"]),
            lr_opacity=float(groups["opacity"]["lr"]), beta1=self.betas[0], beta2=self.betas[1], eps=self.eps,
            grad2d=None if in_registers else ptr(grad2d), radii=None if in_registers else ptr(radii),
            accum=model.xyz_gradient_accum.data_ptr() if want_stats else None,
            denom=model.denom.data_ptr() if want_stats else None,
            max_radii=model.max_radii2D.data_ptr() if want_stats else None)
        a._keep = (gxc, d_scales, d_rots, d_opac, d_nrm, grad2d, radii, sink.saved, sreg)     # (alive until the launch)
        nxt_act = None
        if next_cam is not None:          # (campos [3], R_w2c [3,3], want_normal): the kernel also activates for that camera
            campos, Rn, wn = next_cam
            dev = model._xyz.device
            if campos.is_cuda and Rn.is_cuda and campos.dtype == torch.float32 and Rn.dtype == torch.float32 \
                    and campos.is_contiguous() and Rn.is_contiguous():
                nxt_act = (torch.empty(N, 3, device=dev), torch.empty(N, 4, device=dev), torch.empty(N, 1, device=dev),
                           torch.empty(N, 3, device=dev) if wn else None, torch.empty(N, dtype=torch.uint8, device=dev))
                a.next_campos, a.next_Rw2c = campos.data_ptr(), Rn.data_ptr()
                a.next_scales, a.next_rots, a.next_opac = (t.data_ptr() for t in nxt_act[:3])
                if wn:
                    a.next_normals, a.next_aux = nxt_act[3].data_ptr(), nxt_act[4].data_ptr()

        def commit():
            for k in st:
                st[k]["step"] = nxt[k]
            model._xyz.grad = None
            model._act_cache = None if nxt_act is None else ActivationCache(model, next_cam[0], next_cam[1], next_cam[2], nxt_act)

        return a, commit

    @torch.no_grad()
    def geometry_step(self, model, sink, grad2d=None, radii=None, next_cam=None, normals_world=False):
        """The static tail of an iteration in ONE launch (`vcr_geometry_step`): adjoint of the fused activation + l1_scale
        gradient (from `sink`) -> densification statistics (`grad2d` [N,3] = `means2D_densify.grad`, `radii`; None = skip)
        -> Adam on xyz / scaling / rotation / opacity.  Same arithmetic as activate-backward + `add_densification_stats` +
        `step()` on those groups; their `.grad` must not be set elsewhere (`_xyz.grad` is consumed and cleared here)."""
        if model._xyz.shape[0] == 0:
            return
        a, commit = self.prepare_geometry_step(model, sink, grad2d, radii, next_cam=next_cam, normals_world=normals_world)
        _lib.check(_lib.load().vcr_geometry_step(C.byref(a), _lib.stream_of(model._xyz)))
        commit()

    @torch.no_grad()
    def step_sh_from_rgb(self, drgb, dirs, sh_degree, stream=None):
        """Adam on the f_dc / f_rest groups with the SH gradient formed on the fly as basis(dirs) x drgb (single-view
        training, HIP kernel vcr_sh_adam_from_rgb), launched on `stream` (a torch.cuda.Stream; default: current)."""
        lib = _lib.load()
        groups = {g["name"]: g for g in self.param_groups}
        dc, rest = groups["f_dc"], groups["f_rest"]
        sd, sr = self._state(dc), self._state(rest)
        sd["step"] += 1
        sr["step"] += 1
        if sd["step"] != sr["step"]:
            raise RuntimeError("f_dc / f_rest Adam steps diverged")
        pd, pr = dc["params"][0], rest["params"][0]
        if pd.numel() == 0:
            return
        st = (stream.cuda_stream if stream is not None else torch.cuda.current_stream(pd.device).cuda_stream)
        _lib.check(lib.vcr_sh_adam_from_rgb(pd.shape[0], int(sh_degree), dirs.data_ptr(), drgb.data_ptr(), pd.data_ptr(),
                                            pr.data_ptr(), sd["exp_avg"].data_ptr(), sd["exp_avg_sq"].data_ptr(),
                                            sr["exp_avg"].data_ptr(), sr["exp_avg_sq"].data_ptr(), float(dc["lr"]),
                                            float(rest["lr"]), self.betas[0], self.betas[1], self.eps, int(sd["step"]),
                                            float(self.grad_scale), st))

    @torch.no_grad()
    def step_sh_from_rgb_views(self, drgb_all, xyz, campos_all, sh_degree, stream=None):
        """Data-parallel form of `step_sh_from_rgb`: gradient = sum over views of basis(normalize(xyz - campos_v)) x
        drgb_all[v], times `grad_scale` (HIP kernel vcr_sh_adam_from_rgb_views); `xyz` are the means the views were
        rendered with (a snapshot when the geometry update is already queued)."""
        lib = _lib.load()
        groups = {g["name"]: g for g in self.param_groups}
        dc, rest = groups["f_dc"], groups["f_rest"]
        sd, sr = self._state(dc), self._state(rest)
        sd["step"] += 1
        sr["step"] += 1
        if sd["step"] != sr["step"]:
            raise RuntimeError("f_dc / f_rest Adam steps diverged")
        pd, pr = dc["params"][0], rest["params"][0]
        if pd.numel() == 0:
            return
        st = (stream.cuda_stream if stream is not None else torch.cuda.current_stream(pd.device).cuda_stream)
        _lib.check(lib.vcr_sh_adam_from_rgb_views(pd.shape[0], int(sh_degree), int(drgb_all.shape[0]), xyz.data_ptr(),
                                                  campos_all.data_ptr(), drgb_all.data_ptr(), pd.data_ptr(), pr.data_ptr(),
                                                  sd["exp_avg"].data_ptr(), sd["exp_avg_sq"].data_ptr(), sr["exp_avg"].data_ptr(),
                                                  sr["exp_avg_sq"].data_ptr(), float(dc["lr"]), float(rest["lr"]), self.betas[0],
                                                  self.betas[1], self.eps, int(sd["step"]), float(self.grad_scale), st))

    @torch.no_grad()
    def make_sh_update(self, drgb, sh_degree, view_dirs=None, xyz=None, campos_all=None):
        """The same update as `step_sh_from_rgb` (view_dirs given) / `step_sh_from_rgb_views` (xyz + campos_all given),
        packaged as a `VcrShUpdate` for `VcrRasterArgs.sh_update`: the rasterizer applies it on its colour stream fused
        with the SH -> RGB evaluation of the next forward.  Advances the step counters.  Returns (struct, keep-alive)."""
        groups = {g["name"]: g for g in self.param_groups}
        dc, rest = groups["f_dc"], groups["f_rest"]
        sd, sr = self._state(dc), self._state(rest)
        sd["step"] += 1
        sr["step"] += 1
        if sd["step"] != sr["step"]:
            raise RuntimeError("f_dc / f_rest Adam steps diverged")
        views = 0 if view_dirs is not None else int(drgb.shape[0])
        u = _lib.VcrShUpdate(nviews=views, sh_degree=int(sh_degree), step=int(sd["step"]), grad_scale=float(self.grad_scale),
                             view_dirs=None if view_dirs is None else view_dirs.data_ptr(), drgb=drgb.data_ptr(),
                             xyz=None if xyz is None else xyz.data_ptr(),
                             campos_all=None if campos_all is None else campos_all.data_ptr(),
                             m_dc=sd["exp_avg"].data_ptr(), v_dc=sd["exp_avg_sq"].data_ptr(), m_rest=sr["exp_avg"].data_ptr(),
                             v_rest=sr["exp_avg_sq"].data_ptr(), lr_dc=float(dc["lr"]), lr_rest=float(rest["lr"]),
                             beta1=self.betas[0], beta2=self.betas[1], eps=self.eps)
        return u, (drgb, view_dirs, xyz, campos_all, sd["exp_avg"], sd["exp_avg_sq"], sr["exp_avg"], sr["exp_avg_sq"])

    def zero_grad(self, set_to_none=True):
        for g in self.param_groups:
            for p in g["params"]:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    p.grad.zero_()

    # ---- checkpoint wire format: `torch.optim.Adam.state_dict()` layout (`scene/gaussian_model.py:88-123` stores it in
    # `capture()`, `trainer.py:170-172,425-430` writes / reads `chkpntN.pth`).  `state` is keyed by the parameter's running
    # index over all groups, `step` is a float32 scalar tensor, every group lists its `params` indices and carries torch's
    # hyper-parameter keys; the 1x1-conv classifier is ONE group named "classifier" with two parameters there, kept here
    # as two single-tensor groups "classifier.weight" / "classifier.bias" and merged / split on the way out / in. ----
    @staticmethod
    def _wire_name(name):
        return name.split(".", 1)[0] if name.startswith("classifier.") else name

    @staticmethod
    def _keyed_by_name(sd):
        """Older files of this repo: state keyed by group name, groups without `params`."""
        return any("params" not in g for g in sd["param_groups"]) or not all(isinstance(k, int) for k in sd["state"])

    def state_dict(self):
        template = torch.optim.Adam([torch.zeros(1)], lr=0.0, eps=self.eps, betas=self.betas).param_groups[0]
        state, groups, idx = {}, [], 0
        for g in self.param_groups:
            wire = self._wire_name(g["name"])
            if groups and groups[-1]["name"] == wire:          # second tensor of the classifier group
                wg = groups[-1]
            else:
                wg = {k: v for k, v in template.items() if k != "params"}
                wg.update(lr=g["lr"], name=wire, params=[])
                groups.append(wg)
            wg["params"].append(idx)
            st = self.state.get(g["name"])
            if st is not None:
                state[idx] = dict(step=torch.tensor(float(st["step"])), exp_avg=st["exp_avg"], exp_avg_sq=st["exp_avg_sq"])
            idx += 1
        return dict(state=state, param_groups=groups)

    def load_state_dict(self, sd):
        """Accepts what the reference's `torch.optim.Adam.state_dict()` holds (and, for older files of this repo, the
        name-keyed form).  Groups are matched by name; moments land on the device of the parameter they belong to."""
        if any(not v["exp_avg"].dtype.is_floating_point for v in sd["state"].values() if "exp_avg" in v):
            raise ValueError("optimizer state holds 8-bit codes of GaussianAdamW: load it with optim.optimizer = \"adamw\"")
        by_wire = {}
        for g in self.param_groups:
            by_wire.setdefault(self._wire_name(g["name"]), []).append(g)
        self.state = {}
        if self._keyed_by_name(sd):
            mine = {g["name"]: g for g in self.param_groups}
            for k, v in sd["state"].items():
                if k not in mine:
                    continue
                p = mine[k]["params"][0]
                if tuple(v["exp_avg"].shape) != tuple(p.shape):
                    raise ValueError(f"optimizer state of {k!r} has shape {tuple(v['exp_avg'].shape)}, parameter {tuple(p.shape)}")
                mv = lambda t: t.detach().to(device=p.device, dtype=torch.float32).contiguous()
                self.state[k] = dict(step=int(round(float(v["step"]))), exp_avg=mv(v["exp_avg"]), exp_avg_sq=mv(v["exp_avg_sq"]))
            lrs = {g["name"]: g["lr"] for g in sd["param_groups"]}
            for g in self.param_groups:
                g["lr"] = float(lrs.get(g["name"], g["lr"]))
            return
        for wg in sd["param_groups"]:
            mine = by_wire.get(wg.get("name"))
            if mine is None:
                continue                                       # (e.g. the appearance network: not part of this model)
            if len(mine) != len(wg["params"]):
                raise ValueError(f"optimizer group {wg.get('name')!r}: {len(wg['params'])} tensors saved, {len(mine)} here")
            for g, i in zip(mine, wg["params"]):
                g["lr"] = float(wg["lr"])
                st = sd["state"].get(i)
                if st is None:
                    continue
                p = g["params"][0]
                if tuple(st["exp_avg"].shape) != tuple(p.shape):
                    raise ValueError(f"optimizer state of {g['name']!r} has shape {tuple(st['exp_avg'].shape)}, "
                                     f"parameter {tuple(p.shape)}")
                mv = lambda t: t.detach().to(device=p.device, dtype=torch.float32).contiguous()
                self.state[g["name"]] = dict(step=int(round(float(st["step"]))), exp_avg=mv(st["exp_avg"]),
                                             exp_avg_sq=mv(st["exp_avg_sq"]))


class GaussianAdamW(AdamW):
    """`optim.AdamW` on the Gaussian model's groups, with `FusedAdam`'s checkpoint format: state by running index, groups matched by
    name, the classifier's two tensors as one group -- so checkpoints of either optimizer (and the reference's) load into the
    other's model; 8-bit moments are written as codes and read by this class only."""

    def state_dict(self):
        sd, groups = super().state_dict(), []
        for wg in sd["param_groups"]:
            wg["name"] = FusedAdam._wire_name(wg["name"])
            if groups and groups[-1]["name"] == wg["name"]:
                groups[-1]["params"] += wg["params"]
            else:
                groups.append(wg)
        return dict(state=sd["state"], param_groups=groups)

    def load_state_dict(self, sd):
        """Takes the learning rates and moments of the groups that the file has; the other hyper-parameters are the configuration's.
        Reads what `FusedAdam.load_state_dict` reads."""
        if FusedAdam._keyed_by_name(sd):
            lrs = {wg["name"]: float(wg["lr"]) for wg in sd["param_groups"]}
            names = [g["name"] for g in self.param_groups]
            groups = [dict(params=[i], **(dict(lr=lrs[k]) if k in lrs else {})) for i, k in enumerate(names)]
            state = {i: sd["state"][k] for i, k in enumerate(names) if k in sd["state"]}
            return super().load_state_dict(dict(state=state, param_groups=groups))
        saved = {wg.get("name"): wg for wg in sd["param_groups"]}
        taken, state, groups = {}, {}, []
        for i, g in enumerate(self.param_groups):
            wire = FusedAdam._wire_name(g["name"])
            wg, j = saved.get(wire), taken.get(wire, 0)
            taken[wire] = j + 1
            if wg is None:
                groups.append(dict(params=[i]))
                continue
            if j >= len(wg["params"]):
                raise ValueError(f"optimizer group {wire!r}: {len(wg['params'])} tensors saved, more here")
            self._check_saved(wg)
            groups.append(dict(params=[i], lr=float(wg["lr"])))
            if wg["params"][j] in sd["state"]:
                state[i] = sd["state"][wg["params"][j]]
        for wire, n in taken.items():
            if wire in saved and len(saved[wire]["params"]) != n:
                raise ValueError(f"optimizer group {wire!r}: {len(saved[wire]['params'])} tensors saved, {n} here")
        super().load_state_dict(dict(state=state, param_groups=groups))


class GaussianModel:
    def __init__(self, cfg):
        self.active_sh_degree = 0
        self.max_sh_degree = cfg.sh_degree
        self._xyz = self._features_dc = self._features_rest = torch.empty(0)
        self._scaling = self._rotation = self._opacity = self._objects_dc = torch.empty(0)
        self.max_radii2D = self.xyz_gradient_accum = self.denom = torch.empty(0)
        self.optimizer = None
        self.percent_dense = 0
        self.large_percent_dense = None
        self.spatial_lr_scale = 0
        self.max_mem = getattr(cfg, "max_mem", 22)
        self.enable_semantic = bool(getattr(cfg, "enable_semantic", False))
        self.ch_sem_feat = getattr(cfg, "ch_sem_feat", 0)
        self.num_cls = getattr(cfg, "num_cls", 0)
        self.classifier = None
        self.extent = 1.0
        self.trans = torch.zeros(3)
        self.scale = torch.ones(3)

    # ---- construction --------------------------------------------------------------------------
    def create_from_params(self, raw, spatial_lr_scale, device="cuda"):
        """Initialise from a dict in the reference's storage layout (synthetic.make_gaussians);
        stands in for `create_from_pcd` (`scene/gaussian_model.py:199-229`), whose simple-knn
        dependency is outside the hot path."""
        self.spatial_lr_scale = spatial_lr_scale
        mk = lambda t: torch.nn.Parameter(t.detach().float().to(device).contiguous().requires_grad_(True))
        self._xyz, self._features_dc, self._features_rest = mk(raw["xyz"]), mk(raw["f_dc"]), mk(raw["f_rest"])
        self._scaling, self._rotation, self._opacity = mk(raw["scaling"]), mk(raw["rotation"]), mk(raw["opacity"])
        if "obj_dc" in raw:
            self.enable_semantic = True
            self._objects_dc = mk(raw["obj_dc"])
            self.ch_sem_feat = raw["obj_dc"].shape[-1]
            self.num_cls = self.num_cls or 2
            self.classifier = torch.nn.Conv2d(self.ch_sem_feat, self.num_cls, kernel_size=1).to(device)
        self.max_radii2D = torch.zeros(self._xyz.shape[0], device=device)
        self.trans = self.trans.to(device)
        self.scale = self.scale.to(device)

    def create_from_pcd(self, points, colors, spatial_lr_scale, device="cuda"):
        """`scene/gaussian_model.py:199-229`: isotropic Gaussians at the SfM points, scale = sqrt(mean squared 3-NN
        distance) (HIP `vcr_knn3_mean_dist2` replaces simple-knn's `distCUDA2`), identity rotation, opacity 0.1,
        SH DC from the point colours."""
        from .sh_utils import RGB2SH
        lib = _lib.load()
        pts = torch.as_tensor(points, dtype=torch.float32, device=device).contiguous()
        col = torch.as_tensor(colors, dtype=torch.float32, device=device)
        n = pts.shape[0]
        dist2 = torch.empty(n, device=device)
        _lib.check(lib.vcr_knn3_mean_dist2(n, pts.data_ptr(), dist2.data_ptr(), _lib.stream_of(pts)))
        dist2 = torch.clamp_min(dist2, 0.0000001)
        K = (self.max_sh_degree + 1) ** 2
        rot = torch.zeros(n, 4, device=device)
        rot[:, 0] = 1
        raw = dict(xyz=pts, f_dc=RGB2SH(col)[:, None, :], f_rest=torch.zeros(n, K - 1, 3, device=device),
                   scaling=torch.log(torch.sqrt(dist2))[..., None].repeat(1, 3), rotation=rot,
                   opacity=inverse_sigmoid(0.1 * torch.ones(n, 1, device=device)))
        if self.enable_semantic and self.ch_sem_feat:
            raw["obj_dc"] = RGB2SH(torch.rand(n, 1, self.ch_sem_feat, device=device))
        self.create_from_params(raw, spatial_lr_scale, device=device)

    # ---- getters (scene/gaussian_model.py:125-195) -----------------------------------------------
    @property
    def device(self):
        return self._xyz.device

    @property
    def get_xyz(self):
        return self._xyz

    @property
    def get_scaling(self):
        return torch.exp(self._scaling)

    @property
    def get_rotation(self):
        return torch.nn.functional.normalize(self._rotation)

    @property
    def get_opacity(self):
        return torch.sigmoid(self._opacity)

    @property
    def get_features(self):
        return torch.cat((self._features_dc, self._features_rest), dim=1)

    @property
    def get_objects(self):
        return self._objects_dc

    def get_normal(self, valid=None, idx=None, refine_sign=True, is_all=False):
        """World-space shortest-axis normal (`scene/gaussian_model.py:168-192`): column `argmin(scale)` of the rotation.
        `valid` None + `is_all=False` (the reference's default): rows outside the normalised bounding box stay zero.
        Off the hot path -- `render()` uses `fused_activate`, which also orients and rotates the normal."""
        fill = valid is None and not is_all
        if valid is None:
            valid = (torch.ones(self._xyz.shape[0], dtype=torch.bool, device=self.device) if is_all
                     else self.get_inside_gaus_normalized()[0])
        rot, scaling = self.get_rotation[valid], self.get_scaling[valid]
        if idx is not None:
            rot, scaling = rot[idx], scaling[idx]
        axis = torch.argmin(scaling, dim=-1)
        normals = build_rotation(rot).gather(2, axis[:, None, None].expand(-1, 3, -1)).squeeze(-1)
        if fill:
            out = torch.zeros_like(self._xyz)
            out[valid] = normals
            return out
        return normals

    def get_covariance(self, scaling_modifier=1):
        L = build_rotation(self._rotation) * (scaling_modifier * self.get_scaling)[:, None, :]
        S = L @ L.transpose(1, 2)
        return torch.stack([S[:, 0, 0], S[:, 0, 1], S[:, 0, 2], S[:, 1, 1], S[:, 1, 2], S[:, 2, 2]], 1)

    def get_inside_gaus_normalized(self):
        """`tools/math_utils.py:50-74` with a translation-vector `trans`."""
        pts = (self._xyz - self.trans) / self.scale
        with torch.no_grad():
            inside = torch.all(torch.abs(pts) < 1, dim=-1)
        return inside, pts

    def oneupSHdegree(self):
        if self.active_sh_degree < self.max_sh_degree:
            self.active_sh_degree += 1

    # ---- optimiser (scene/gaussian_model.py:232-270) -----------------------------------------------
    def _param_table(self):
        t = {"xyz": "_xyz", "f_dc": "_features_dc", "f_rest": "_features_rest", "opacity": "_opacity",
             "scaling": "_scaling", "rotation": "_rotation"}
        if self.enable_semantic:
            t["obj_dc"] = "_objects_dc"
        return t

    def training_setup(self, training_args):
        self.percent_dense = training_args.percent_dense
        dl = getattr(training_args, "densify_large", None)
        self.large_percent_dense = dl.percent_dense if (dl is not None and getattr(dl, "percent_dense", 0) > 0) else None
        N, dev = self._xyz.shape[0], self.device
        self.xyz_gradient_accum = torch.zeros((N, 1), device=dev)
        self.denom = torch.zeros((N, 1), device=dev)
        lrs = {"xyz": training_args.position_lr_init * self.spatial_lr_scale, "f_dc": training_args.feature_lr,
               "f_rest": training_args.feature_lr / 20.0, "opacity": training_args.opacity_lr,
               "scaling": training_args.scaling_lr, "rotation": training_args.rotation_lr,
               "obj_dc": training_args.feature_lr}
        groups = [{"params": [getattr(self, attr)], "lr": lrs[name], "name": name}
                  for name, attr in self._param_table().items()]
        if self.enable_semantic and self.classifier is not None:
            # `scene/gaussian_model.py:254`: the 1x1-conv classifier trains with Adam at cls_lr.  Not per-Gaussian, so the
            # groups are flagged "aux": densify / prune surgery skips them (`:428,445,483`); the DP bucket includes them.
            for pn, prm in self.classifier.named_parameters():
                groups.append({"params": [prm], "lr": getattr(training_args, "cls_lr", 5e-4), "name": "classifier." + pn,
                               "aux": True})
        kind = getattr(training_args, "optimizer", "adam")
        if kind == "adam":
            if getattr(training_args, "max_grad_norm", None) or float(getattr(training_args, "weight_decay", 0.0)) or \
                    int(getattr(training_args, "state_bits", 32)) != 32:
                raise ValueError("optim.max_grad_norm, weight_decay and state_bits need optim.optimizer = \"adamw\"")
            self.optimizer = FusedAdam(groups, eps=1e-15)
        elif kind == "adamw":
            self.optimizer = GaussianAdamW(groups, eps=1e-15, weight_decay=float(getattr(training_args, "weight_decay", 0.0)),
                                           state_bits=int(getattr(training_args, "state_bits", 32)))
        else:
            raise ValueError(f"optim.optimizer = {kind!r}: \"adam\" or \"adamw\"")
        self.xyz_scheduler_args = get_expon_lr_func(
            lr_init=training_args.position_lr_init * self.spatial_lr_scale,
            lr_final=training_args.position_lr_final * self.spatial_lr_scale,
            lr_delay_mult=training_args.position_lr_delay_mult, max_steps=training_args.position_lr_max_steps)

    def update_learning_rate(self, iteration):
        for g in self.optimizer.param_groups:
            if g["name"] == "xyz":
                g["lr"] = float(self.xyz_scheduler_args(iteration))
                return g["lr"]

    # ---- densification statistics --------------------------------------------------------------------
    @torch.no_grad()
    def add_densification_stats(self, viewspace_point_tensor, update_filter=None, radii=None):
        """`scene/gaussian_model.py:669-671` (+ the max_radii2D update of `trainer.py:345` when `radii`
        is given): one HIP kernel instead of three masked index ops."""
        g = viewspace_point_tensor.grad if viewspace_point_tensor.grad is not None else viewspace_point_tensor
        if radii is None:
            self.xyz_gradient_accum[update_filter] += torch.norm(g[update_filter, :2], dim=-1, keepdim=True)
            self.denom[update_filter] += 1
            return
        lib = _lib.load()
        g = g.contiguous()
        _lib.check(lib.vcr_densify_stats(g.shape[0], g.data_ptr(), radii.data_ptr(), self.xyz_gradient_accum.data_ptr(),
                                         self.denom.data_ptr(), self.max_radii2D.data_ptr(), _lib.stream_of(g)))

    # ---- optimiser-state surgery (scene/gaussian_model.py:425-531) -----------------------------------
    def _moments_of(self, name):
        """-> the two moments of a group as float32 tensors, or None if it has none yet."""
        st = self.optimizer.state.get(name)
        if st is None:
            return None
        if isinstance(self.optimizer, AdamW):
            return self.optimizer.moments_of(name)
        return st["exp_avg"], st["exp_avg_sq"]

    def _store_moments(self, name, m, v):
        """The group's parameter has been replaced: these new tensors are its moments now (8 bits: to the nearest code)."""
        if isinstance(self.optimizer, AdamW) and self.optimizer.state_bits == 8:
            self.optimizer.set_moments(name, m, v)
        else:
            self.optimizer.state[name].update(exp_avg=m, exp_avg_sq=v)

    def _set_params(self, new):
        for name, attr in self._param_table().items():
            setattr(self, attr, new[name])

    def _rebind(self, fn_param, fn_state):
        out = {}
        for g in self.optimizer.param_groups:
            if g.get("aux"):
                continue
            p = g["params"][0]
            newp = torch.nn.Parameter(fn_param(g["name"], p.detach()).contiguous().requires_grad_(True))
            mv = self._moments_of(g["name"])
            g["params"][0] = newp
            if mv is not None:
                self._store_moments(g["name"], *(fn_state(g["name"], t).contiguous() for t in mv))
            out[g["name"]] = newp
        self._set_params(out)

    # -- fused row surgery (HIP): every per-Gaussian array of the model moves in ONE launch (csrc/model_ops.hip) ------------
    def _move_rows(self, mask, mode, copies=1, reset_stats=True):
        """mode 0: keep the rows where `mask` (prune); mode 1: append `copies` copies of the rows where `mask` (clone /
        split), Adam moments of the appended rows zero.  Parameters, both moments and the densification statistics are
        re-packed by `vcr_rows_plan` + `vcr_rows_move`, 8-bit moments by `vcr_moments8_rows`; returns the number of selected rows."""
        lib = _lib.load()
        dev, N = self.device, self._xyz.shape[0]
        m8 = mask.to(torch.uint8).contiguous()
        st = _lib.stream_of(m8)
        plan = torch.empty(lib.vcr_rows_plan_bytes(N) // 4, dtype=torch.int32, device=dev)
        _lib.check(lib.vcr_rows_plan(N, m8.data_ptr(), plan.data_ptr(), st))
        M = int(plan[-1])                                   # the one host sync (the reference's boolean indexing has the same)
        newN = M if mode == 0 else N + copies * M
        items = []                                          # (setter, old tensor, zero_new)
        packed = isinstance(self.optimizer, AdamW) and self.optimizer.state_bits == 8
        for g in self.optimizer.param_groups:
            if g.get("aux"):
                continue
            items.append((("p", g), g["params"][0].detach(), False))
            if packed:                                      # (8-bit moments move as codes, below)
                continue
            mv = self._moments_of(g["name"])
            if mv is not None:
                items.append((("m", g["name"]), mv[0], True))
                items.append((("v", g["name"]), mv[1], True))
        keep_stats = mode == 0 or not reset_stats
        if keep_stats:
            items += [(("s", "xyz_gradient_accum"), self.xyz_gradient_accum, True), (("s", "denom"), self.denom, True),
                      (("s", "max_radii2D"), self.max_radii2D, True)]
        arr = _lib.VcrRowArrays()
        outs = []
        for k, (_, t, zero_new) in enumerate(items):
            t = t.contiguous()
            out = torch.empty((newN,) + tuple(t.shape[1:]), dtype=torch.float32, device=dev)
            width = 1
            for d in t.shape[1:]:
                width *= int(d)
            arr.a[k].inp, arr.a[k].out, arr.a[k].width, arr.a[k].zero_new = t.data_ptr(), out.data_ptr(), width, int(zero_new)
            outs.append((t, out))
        arr.n = len(items)
        _lib.check(lib.vcr_rows_move(N, m8.data_ptr(), plan.data_ptr(), C.byref(arr), mode, copies, st))
        new_params, moved = {}, {}
        for (kind, ref), (_, out) in zip([it[0] for it in items], outs):
            if kind == "p":
                ref["params"][0] = torch.nn.Parameter(out.requires_grad_(True))
                new_params[ref["name"]] = ref["params"][0]
            elif kind == "m":
                moved[ref] = out
            elif kind == "v":
                self._store_moments(ref, moved[ref], out)
            else:
                setattr(self, ref, out)
        self._set_params(new_params)
        held = [self.optimizer.state[n] for n in new_params if n in self.optimizer.state] if packed else []
        if held:
            index = m8.nonzero().view(-1).int() if mode == 0 else torch.cat(
                (torch.arange(N, dtype=torch.int32, device=dev), torch.full((copies * M,), -1, dtype=torch.int32, device=dev)))
            for st8, new in zip(held, rows8(held, index)):
                st8.update(new)
        if not keep_stats:
            self.xyz_gradient_accum = torch.zeros((newN, 1), device=dev)
            self.denom = torch.zeros((newN, 1), device=dev)
            self.max_radii2D = torch.zeros(newN, device=dev)
        return M

    @torch.no_grad()
    def prune_points(self, mask):
        """`scene/gaussian_model.py:456-475`."""
        if self._xyz.is_cuda:
            self._move_rows(~mask, 0)
            return
        keep = ~mask                  # host tensors (CPU unit tests of the surgery logic): plain indexing
        self._rebind(lambda n, p: p[keep], lambda n, s: s[keep])
        self.xyz_gradient_accum = self.xyz_gradient_accum[keep]
        self.denom = self.denom[keep]
        self.max_radii2D = self.max_radii2D[keep]

    @torch.no_grad()
    def densification_postfix(self, new, reset=True):
        """`scene/gaussian_model.py:495-531` for explicitly given new rows (`new`: {group: tensor})."""
        self._rebind(lambda n, p: torch.cat((p, new[n]), 0), lambda n, s: torch.cat((s, torch.zeros_like(new[n])), 0))
        N, dev = self._xyz.shape[0], self.device
        if reset:
            self.xyz_gradient_accum = torch.zeros((N, 1), device=dev)
            self.denom = torch.zeros((N, 1), device=dev)
            self.max_radii2D = torch.zeros(N, device=dev)
        else:
            k = N - self.max_radii2D.shape[0]
            self.xyz_gradient_accum = torch.cat((self.xyz_gradient_accum, torch.zeros((k, 1), device=dev)))
            self.denom = torch.cat((self.denom, torch.zeros((k, 1), device=dev)))
            self.max_radii2D = torch.cat((self.max_radii2D, torch.zeros(k, device=dev)))

    def _gather(self, mask, times=1):
        out = {}
        for name, attr in self._param_table().items():
            v = getattr(self, attr).detach()[mask]
            out[name] = torch.cat([v] * times, 0) if times > 1 else v
        return out

    def _append_selected(self, sel, copies=1):
        """cat(rows, rows[sel] x copies) for every array (moments of the new rows zero, statistics reset)."""
        if self._xyz.is_cuda:
            return self._move_rows(sel, 1, copies=copies, reset_stats=True)
        self.densification_postfix(self._gather(sel, times=copies))
        return int(sel.sum())

    @torch.no_grad()
    def densify_and_clone(self, grads, grad_threshold, scene_extent):
        sel = torch.norm(grads, dim=-1) >= grad_threshold
        sel &= self.get_scaling.max(dim=1).values <= self.percent_dense * scene_extent
        self._append_selected(sel)

    @torch.no_grad()
    def densify_and_split_along_maxscaling(self, grads, grad_threshold, scene_extent, visi=None, N=2, n_std=2):
        """Deterministic two-way split along the longest axis (`scene/gaussian_model.py:579-628`):
        children at mu +- (n_std/3) s_max e_max, longest scale divided by 0.8 N."""
        n0 = self._xyz.shape[0]
        padded = torch.zeros(n0, device=self.device)
        padded[:grads.shape[0]] = grads.squeeze()
        smax = self.get_scaling.max(dim=1).values
        sel = (padded >= grad_threshold) & (smax > self.percent_dense * scene_extent)
        mem_gb = torch.cuda.memory_allocated(self.device) / 1024 ** 3 if self.device.type == "cuda" else 0.0
        if self.large_percent_dense is not None and mem_gb < self.max_mem:
            big = (smax > self.large_percent_dense * scene_extent) & self.get_inside_gaus_normalized()[0]
            if visi is not None:
                pv = torch.zeros(n0, device=self.device, dtype=torch.bool)
                pv[:visi.shape[0]] = visi
                big &= pv
            sel |= big
        scaling = self.get_scaling[sel]
        rots = build_rotation(self._rotation.detach()[sel])
        axis = torch.argmax(scaling, dim=-1)
        ar = torch.arange(scaling.shape[0], device=self.device)
        max_s = scaling[ar, axis]
        dirs = rots.gather(2, axis[:, None, None].expand(-1, 3, -1)).squeeze(-1)
        off = dirs * (n_std * max_s / 3.0)[:, None]
        base = self._xyz.detach()[sel]
        ns = scaling.clone()
        ns[ar, axis] = max_s / (0.8 * N)
        # all arrays: two copies of the selected rows appended; then the children's means / log-scales overwrite theirs
        self._append_selected(sel, copies=N)
        self._xyz.data[n0:] = torch.cat((base + off, base - off), 0)
        self._scaling.data[n0:] = torch.log(ns).repeat(N, 1)
        prune = torch.cat((sel, torch.zeros(self._xyz.shape[0] - n0, device=self.device, dtype=torch.bool)))
        self.prune_points(prune)

    @torch.no_grad()
    def densify_and_prune(self, max_grad, min_opacity, extent, max_screen_size, visi=None):
        """`scene/gaussian_model.py:643-659`."""
        grads = self.xyz_gradient_accum / self.denom
        grads[grads.isnan()] = 0.0
        self.densify_and_clone(grads, max_grad, extent)
        self.densify_and_split_along_maxscaling(grads, max_grad, extent, visi=visi)
        prune = (self.get_opacity < min_opacity).squeeze()
        if max_screen_size:
            prune |= self.max_radii2D > max_screen_size
            prune |= self.get_scaling.max(dim=1).values > 0.1 * extent
        self.prune_points(prune)

    @torch.no_grad()
    def reset_opacity(self):
        """`scene/gaussian_model.py:361-364`: opacity <- min(opacity, 0.01), Adam moments zeroed."""
        new = inverse_sigmoid(torch.min(self.get_opacity, torch.ones_like(self.get_opacity) * 0.01))
        for g in self.optimizer.param_groups:
            if g["name"] == "opacity":
                g["params"][0] = torch.nn.Parameter(new.contiguous().requires_grad_(True))
                if self.optimizer.state.get("opacity") is not None:
                    self._store_moments("opacity", torch.zeros_like(new), torch.zeros_like(new))
                self._opacity = g["params"][0]

    @torch.no_grad()
    def prune_gaussians(self, percent, import_score):
        """`scene/gaussian_model.py:661-667`."""
        s, _ = torch.sort(import_score, dim=0)
        thr = s[int(percent * (s.shape[0] - 1))]
        self.prune_points((import_score <= thr).squeeze())

    # ---- PLY wire format (scene/gaussian_model.py:272-320,366-423): binary little-endian, all-f4 vertex element
    def construct_list_of_attributes(self):
        l = ["x", "y", "z", "nx", "ny", "nz"]
        l += [f"f_dc_{i}" for i in range(self._features_dc.shape[1] * self._features_dc.shape[2])]
        l += [f"f_rest_{i}" for i in range(self._features_rest.shape[1] * self._features_rest.shape[2])]
        l += ["opacity"] + [f"scale_{i}" for i in range(3)] + [f"rot_{i}" for i in range(4)]
        if self.enable_semantic:
            l += [f"obj_dc_{i}" for i in range(self._objects_dc.shape[1] * self._objects_dc.shape[2])]
        return l

    @torch.no_grad()
    def save_ply(self, path, normals=None):
        """Same fields, order and channel-major SH flattening as the reference's `point_cloud.ply`, so files go
        straight into its viewer / mesh / eval tools.  Written with numpy (plyfile is not a dependency)."""
        import os
        os.makedirs(os.path.dirname(os.path.abspath(path)), exist_ok=True)
        cpu = lambda t: t.detach().float().cpu().numpy()
        xyz = cpu(self._xyz)
        cols = [xyz, np.zeros_like(xyz) if normals is None else cpu(normals),
                cpu(self._features_dc.transpose(1, 2).flatten(start_dim=1)),
                cpu(self._features_rest.transpose(1, 2).flatten(start_dim=1)), cpu(self._opacity), cpu(self._scaling),
                cpu(self._rotation)]
        if self.enable_semantic:
            cols.append(cpu(self._objects_dc.transpose(1, 2).flatten(start_dim=1)))
        data = np.ascontiguousarray(np.concatenate(cols, axis=1).astype("<f4"))
        names = self.construct_list_of_attributes()
        assert data.shape[1] == len(names)
        header = "ply\nformat binary_little_endian 1.0\nelement vertex %d\n" % data.shape[0]
        header += "".join(f"property float {n}\n" for n in names) + "end_header\n"
        with open(path, "wb") as f:
            f.write(header.encode("ascii"))
            f.write(data.tobytes())

    def load_ply(self, path, device="cuda"):
        with open(path, "rb") as f:
            names, n = [], 0
            line = f.readline().strip()
            assert line == b"ply"
            while True:
                line = f.readline().strip().decode("ascii")
                if line.startswith("element vertex"):
                    n = int(line.split()[-1])
                elif line.startswith("property"):
                    parts = line.split()
                    assert parts[1] in ("float", "float32"), "only all-float vertex elements are supported"
                    names.append(parts[2])
                elif line.startswith("format"):
                    assert "binary_little_endian" in line
                elif line == "end_header":
                    break
            data = np.frombuffer(f.read(4 * n * len(names)), dtype="<f4").reshape(n, len(names))
        col = {nm: i for i, nm in enumerate(names)}
        pick = lambda keys: torch.from_numpy(np.stack([data[:, col[k]] for k in keys], 1).copy())
        srt = lambda pre: sorted([k for k in names if k.startswith(pre)], key=lambda k: int(k.split("_")[-1]))
        K = (self.max_sh_degree + 1) ** 2
        rest = srt("f_rest_")
        assert len(rest) == 3 * (K - 1), "PLY SH degree does not match the model"
        mk = lambda t: torch.nn.Parameter(t.float().to(device).contiguous().requires_grad_(True))
        self._xyz = mk(pick(["x", "y", "z"]))
        self._features_dc = mk(pick(srt("f_dc_")).reshape(n, 3, 1).transpose(1, 2))
        self._features_rest = mk(pick(rest).reshape(n, 3, K - 1).transpose(1, 2))
        self._opacity = mk(pick(["opacity"]))
        self._scaling = mk(pick(srt("scale_")))
        self._rotation = mk(pick(srt("rot_")))
        obj = srt("obj_dc_")
        if obj:
            self.enable_semantic = True
            self.ch_sem_feat = len(obj)
            self._objects_dc = mk(pick(obj).reshape(n, len(obj), 1).transpose(1, 2))
        self.max_radii2D = torch.zeros(n, device=device)
        self.active_sh_degree = self.max_sh_degree

    # ---- checkpoint (scene/gaussian_model.py:88-123) ---------------------------------------------------
    def capture(self):
        return (self.active_sh_degree, self._xyz, self._features_dc, self._features_rest, self._scaling, self._rotation,
                self._opacity, self._objects_dc, self.max_radii2D, self.xyz_gradient_accum, self.denom,
                self.optimizer.state_dict(), self.spatial_lr_scale)

    def restore(self, model_args, training_args, device=None):
        """`scene/gaussian_model.py:102-123`.  `model_args` is the tuple of `capture()` -- this repo's or the reference's
        (the first element of a `chkpntN.pth`, `trainer.py:170-172`); `device`: where the model shall live (default: where
        the checkpoint's tensors are)."""
        (self.active_sh_degree, xyz, f_dc, f_rest, scaling, rotation, opacity, obj_dc, radii, acc, den, opt,
         self.spatial_lr_scale) = model_args
        dev = torch.device(device) if device is not None else xyz.device
        mk = lambda t: torch.nn.Parameter(t.detach().to(device=dev, dtype=torch.float32).contiguous().requires_grad_(True))
        self._xyz, self._features_dc, self._features_rest = mk(xyz), mk(f_dc), mk(f_rest)
        self._scaling, self._rotation, self._opacity = mk(scaling), mk(rotation), mk(opacity)
        if obj_dc is not None and obj_dc.numel() > 0:
            self.enable_semantic = True
            self._objects_dc = mk(obj_dc)
            self.ch_sem_feat = int(obj_dc.shape[-1])
            fresh_classifier = self.classifier is None
            if fresh_classifier:
                # the classifier's WEIGHTS travel in the reference's model.pth, not in the checkpoint
                # (`scene/gaussian_model.py:304-311`); the checkpoint only holds their Adam moments.  A classifier created
                # here is randomly initialised: its saved moments belong to other weights and are NOT restored.
                if not self.num_cls:
                    raise ValueError("restore(): the checkpoint carries semantic features but the model has no classifier and "
                                     "cfg.num_cls is unset -- load / construct the classifier (model.pth) before restore()")
                import warnings
                warnings.warn("restore(): no classifier loaded before the checkpoint; a randomly initialised one is created and "
                              "its optimizer state in the checkpoint is skipped (load model.pth first to resume semantics)")
                self.classifier = torch.nn.Conv2d(self.ch_sem_feat, self.num_cls, kernel_size=1)
            self.classifier = self.classifier.to(dev)
        else:
            self._objects_dc = torch.empty(0, device=dev)
        self.max_radii2D = radii.detach().to(dev).float()
        self.trans, self.scale = self.trans.to(dev), self.scale.to(dev)
        self.training_setup(training_args)
        self.xyz_gradient_accum, self.denom = acc.detach().to(dev).float(), den.detach().to(dev).float()
        self.optimizer.load_state_dict(opt)
        if obj_dc is not None and obj_dc.numel() > 0 and fresh_classifier:
            for k in ("classifier.weight", "classifier.bias"):
                self.optimizer.state.pop(k, None)
