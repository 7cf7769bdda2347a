"""Host-side mirror of the per-Gaussian update that follows loss.backward() in a VEGS iteration, computed
by fused HIP kernels (vegs_amd/csrc/optim.hip, C ABI include/vegs_optim.h):

  Adam(params, lr, betas, eps)          drop-in for torch.optim.Adam as scene/gaussian_model.py:159-168 builds it
                                        (six named groups, eps=1e-15) and train.py:319-320 steps it
  add_densification_stats(...)          scene/gaussian_model.py:411-413 + the max_radii2D line of train.py:299
  densify_and_prune(optimizer, ...)     scene/gaussian_model.py:384-403 with its clone / split / prune and the
                                        optimizer-state surgery (:278-351), as one planned gather
  reset_opacity(optimizer)              scene/gaussian_model.py:215-218
  grad_norm(parameters) / clip_grad_norm_(parameters, max_norm)
                                        the global norm of many gradients, and torch.nn.utils.clip_grad_norm_
  step_many(optimizers, max_grad_norm)  the Adam step of the clipped gradients, without rewriting them

`Adam` is a torch.optim.Optimizer: param_groups (with the reference's extra "name" keys) and the per-parameter
state dict {"step", "exp_avg", "exp_avg_sq"} have torch's layout, because the reference's densification code
edits them in place (scene/gaussian_model.py:263-331: _prune_optimizer, cat_tensors_to_optimizer,
replace_tensor_to_optimizer) and checkpoints them with state_dict().  One kernel launch updates all groups.
GPU tensors only; there is no CPU path.
"""
import ctypes as C
import math
import struct

import torch

from . import _capi


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False):
        if weight_decay != 0 or amsgrad:
            raise NotImplementedError("the fused Adam covers the reference's configuration: no weight decay, no amsgrad")
        if lr < 0.0 or eps < 0.0 or not (0.0 <= betas[0] < 1.0) or not (0.0 <= betas[1] < 1.0):
            raise ValueError("invalid Adam hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=0, amsgrad=False))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        step_many([self])
        return loss


def _entries(optimizer):
    """[(parameter, gradient, group, its state or None, optimizer)] of one optimizer (vegs_amd.optim.Adam or torch.optim.Adam:
    same state layout), parameters without a gradient left out -- with everything checked WITHOUT touching the optimizer: step_many
    goes through every optimizer of its batch before the first step counter moves, so an exception leaves all of them exactly
    as they were (a half-advanced batch would skew the bias correction of a retry and desynchronise the ranks of a
    distributed job)."""
    out = []
    for group in optimizer.param_groups:
        if group.get("weight_decay", 0) != 0 or group.get("amsgrad", False) or group.get("maximize", False):
            raise NotImplementedError("the fused Adam covers the reference's configuration: no weight decay, no amsgrad")
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            if not p.is_cuda:
                raise ValueError("fused Adam expects GPU parameters (there is no CPU path)")
            if p.dtype != torch.float32 or g.dtype != torch.float32 or g.is_sparse:
                raise ValueError("fused Adam expects dense float32 parameters and gradients")
            if not p.is_contiguous():
                raise ValueError("fused Adam expects contiguous parameters")
            st = optimizer.state.get(p) or None
            if st is not None:
                m, v, shape = st.get("exp_avg"), st.get("exp_avg_sq"), p.shape
                if (m is None or v is None or "step" not in st or m.shape != shape or v.shape != shape
                        or not m.is_contiguous() or not v.is_contiguous()):
                    raise ValueError("optimizer state does not match its parameter")
            out.append((p, g, group, st, optimizer))
    return out


def _advance(step):
    """step += 1 on a state's counter, and its new value as a number."""
    if step.is_cuda or step.dtype != torch.float32:
        step += 1
        return int(step.item())
    n = C.c_float.from_address(step.data_ptr())       # (the tensor's own memory: a third of the time of the addition through torch)
    n.value += 1.0
    return int(n.value)


_ADAM = struct.Struct("4Qqdqd")           # VrAdamTensor


def _written(tensors):
    """Raises the version of tensors that a kernel writes through their addresses, as torch's in-place operations do: a graph
    that still needs the old values raises in its backward instead of computing on with the new ones."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:                              # (inference tensors have none)
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _grads_of(parameters):
    """The gradients of `parameters` -- a tensor, an optimizer, or an iterable of either -- each one once."""
    if isinstance(parameters, (torch.Tensor, torch.optim.Optimizer)):
        parameters = [parameters]
    grads = []
    for p in parameters:
        if isinstance(p, torch.Tensor):
            grads.append(p.grad)
        else:
            grads += [q.grad for group in p.param_groups for q in group["params"]]
    return _once(g for g in grads if g is not None)


def _once(grads):
    """{(address, elements, type): gradient} of gradients that fill their memory, with shape and strides behind these where one does
    not: each one once.  (The order of the dimensions does not tell two that fill the same memory apart, but the strides tell two
    others that begin at one address.)"""
    kinds, seen = _capi.VR_DTYPES, {}
    for g in grads:
        if g.layout is not torch.strided:
            raise ValueError(f"gradients must be dense float32, bfloat16 or float16 tensors (got {g.layout})")
        key = g.data_ptr(), g.numel(), kinds.get(g.dtype, g.dtype)               # (other types are refused by _grad_table)
        if not g.is_contiguous() and not _dense(g):
            key += g.shape, g.stride()
        seen[key] = g
    return seen


def _dense(t):
    """Whether the elements of `t` fill their memory without gaps or repeats, in whatever order (a norm or a scaling does
    not care about the order)."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _grad_table(seen):
    """(flat VrGradTensor words, device, [(gradient, copy of it)]) of what _once returns, checked: gradients that do not fill their
    memory are copied."""
    device = next(iter(seen.values())).device
    if device.type != "cuda" or len({g.get_device() for g in seen.values()}) != 1:
        raise ValueError("gradients to be clipped together must be GPU tensors on one device (there is no CPU path)")
    flat, copies = [], []
    for key, g in seen.items():
        if isinstance(key[2], torch.dtype):
            raise ValueError(f"gradients must be dense float32, bfloat16 or float16 tensors (got {key[2]})")
        if len(key) > 3:
            copy = g.contiguous()
            copies.append((g, copy))
            key = (copy.data_ptr(), key[1], key[2])
        flat += key
    return struct.pack("%dq" % len(flat), *flat), device, copies


def _norm_kind(norm_type):
    norm_type = float(norm_type)
    if norm_type == 2.0:
        return 2
    if norm_type == math.inf:
        return 0
    raise NotImplementedError(f"norm_type {norm_type}: the 2-norm and the largest magnitude (inf) are supported")


def _check_max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN (got {max_norm})")
    return max_norm


def _norm_and_scratch(lib, count, n_factors, near):
    """(a 0-dim float32 tensor, the norm's scratch) on the device of `near`, which is current."""
    return (near.new_empty((), dtype=torch.float32),
            near.new_empty(lib.vr_grad_norm_scratch_bytes(count, n_factors) >> 3, dtype=torch.float64))


def grad_norm(parameters, norm_type=2.0, sh_factors=()):
    """The norm of all gradients of `parameters` (a tensor, an optimizer, or an iterable of either) as if they were one
    vector: a 0-dim float32 tensor on their device.  Squares and sums are taken in 64 bits in an order that depends on the
    sizes only -- every rank that holds the same gradients gets the same bits.  Parameters without a gradient are skipped,
    a gradient met twice counts once; no gradients at all give a zero on the CPU, as in torch.

    norm_type: 2.0 or math.inf (the largest magnitude).  Gradients: float32, bfloat16 or float16.
    sh_factors: gradients that exist only as factors, as (means3D, campos, factors, sh_degree, scale) -- the arguments of
    adam_step_sh_factored, whose gradient enters the norm without being written."""
    kind = _norm_kind(norm_type)
    return _norm_of(_grads_of(parameters), kind, sh_factors)


def _norm_of(seen, kind, sh_factors=()):
    items = []
    table, device, copies = _grad_table(seen) if seen else (None, None, None)
    for means3D, campos, factors, sh_degree, scale in sh_factors:
        P, n, means3D, campos, factors, fstride = _check_factor_inputs(means3D, campos, factors)
        device = device or means3D.device
        if means3D.device != device:
            raise ValueError("gradients to be clipped together must be GPU tensors on one device (there is no CPU path)")
        keep_f = (means3D, campos, factors)
        items.append((_capi.VrShGradFactors(_capi.ptr(means3D), _capi.ptr(campos), _capi.ptr(factors), fstride, P, n,
                                            int(sh_degree), float(scale)), keep_f))
    if not seen and not items:
        return torch.tensor(0.0)
    lib = _capi.load()
    with _capi.on(device):
        norm, scratch = _norm_and_scratch(lib, len(seen), len(items), next(iter(seen.values())) if seen else means3D)
        _capi.check(lib.vr_grad_norm(table, len(seen), (_capi.VrShGradFactors * len(items))(*[i[0] for i in items]) if items else None,
                                     len(items), kind, norm.data_ptr(), scratch.data_ptr(), _capi.stream_of(device)))
    return norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ on the GPU: scales the gradients of `parameters` (a tensor, an optimizer, or an iterable
    of either) in place by min(1, max_norm / (norm + 1e-6)) and returns their norm from before, a 0-dim float32 tensor.
    The norm is grad_norm()'s.  Gradients below the bound are not written at all; a NaN norm makes all of them NaN, as in
    torch.  Two gradients that share a part of their memory are refused, unless the elements of one do not fill their memory:
    then each value in memory is scaled once, and enters the norm once for each gradient that holds it.
    error_if_nonfinite=True waits for the norm and raises before anything is scaled.  `foreach` has no effect (there
    is one path).  step_many(max_grad_norm=...) clips inside the Adam step instead and leaves the gradients alone."""
    max_norm, kind = _check_max_norm(max_norm), _norm_kind(norm_type)
    grads = _grads_of(parameters)
    if not grads:
        return torch.tensor(0.0)
    table, device, copies = _grad_table(grads)
    for g, _ in copies:
        if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
            raise ValueError("an expanded gradient (one value in memory for several elements) cannot be clipped in place")
    lib = _capi.load()
    with _capi.on(device):
        norm, scratch = _norm_and_scratch(lib, len(grads), 0, next(iter(grads.values())))
        stream = _capi.stream_of(device)
        if error_if_nonfinite:
            _capi.check(lib.vr_grad_norm(table, len(grads), None, 0, kind, norm.data_ptr(), scratch.data_ptr(), stream))
            if not math.isfinite(norm.item()):
                raise RuntimeError(f"the total norm of order {float(norm_type)} of the gradients is not finite, so they cannot be "
                                   "clipped; error_if_nonfinite=False scales them all the same")
            _written(list(grads.values()))
            rc = lib.vr_clip_grads(table, len(grads), norm.data_ptr(), max_norm, stream)
        else:
            _written(list(grads.values()))
            rc = lib.vr_clip_grad_norm(table, len(grads), kind, max_norm, norm.data_ptr(), scratch.data_ptr(), stream)
    if rc == _capi.INVALID_ARGUMENT:                  # (what is left for the library to refuse: shared memory)
        raise ValueError(lib.vr_last_error().decode())
    _capi.check(rc)
    for g, copy in copies:
        g.copy_(copy)
    return norm


def _check_norm(norm, device):
    if not isinstance(norm, torch.Tensor) or norm.device != device or norm.dtype != torch.float32 or norm.numel() != 1:
        raise ValueError(f"grad_norm must be a float32 tensor of one value on {device} (what optim.grad_norm returns)")


@torch.no_grad()
def step_many(optimizers, max_grad_norm=None, grad_norm=None):
    """optimizer.step() of SEVERAL Adam optimizers as one launch (per 64 tensors): what train.py:254-275 does one optimizer
    after the other when dynamic objects are in frame -- the static model's six groups, six more per instance model
    (densification_and_optimization(..., box=True)) and the three pose corrections of every BoxModel
    (box_model.optimizer.step(), model/boxmodel.py:13) -- with every tensor's own learning rate, step count and eps in
    the kernel's block->tensor table.  Optimizers may be vegs_amd.optim.Adam or torch.optim.Adam (same state layout).
    All-or-nothing: every optimizer is validated before any state (step counters, fresh moments) is touched.

    max_grad_norm: step with the gradients clipped to this global norm, as if clip_grad_norm_ had been called on all the
    optimizers together before -- but the factor is applied where Adam loads a gradient, and .grad keeps its values.
    Returns the norm (0-dim float32 on the GPU) then.  grad_norm: that norm where the caller has it already, from
    optim.grad_norm over these AND other gradients (one joint norm for several calls)."""
    optimizers = list(optimizers)
    if max_grad_norm is None:
        if grad_norm is not None:
            raise ValueError("grad_norm without max_grad_norm")
    else:
        max_grad_norm = _check_max_norm(max_grad_norm)
    lib = _capi.load()
    batch = [entry for opt in optimizers for entry in _entries(opt)]
    if len({id(entry[0]) for entry in batch}) != len(batch):
        raise ValueError("a parameter is in two of the optimizers, or an optimizer twice in the list: one launch steps each parameter once")
    norm = None
    if max_grad_norm is not None:
        if grad_norm is not None:
            for index in {entry[0].get_device() for entry in batch}:
                _check_norm(grad_norm, torch.device("cuda", index))
        norm = grad_norm if grad_norm is not None else _norm_of(_once([entry[1] for entry in batch]), 2)
    by_cfg, keep, written = {}, [], []
    for p, g, group, st, opt in batch:
        if st is None:
            st = opt.state[p]
            if len(st) == 0:
                st["step"] = torch.tensor(0.0, dtype=torch.float32)
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        b1, b2 = group["betas"]
        m, v = st["exp_avg"], st["exp_avg_sq"]
        written += (p, m, v)
        by_cfg.setdefault((p.get_device(), float(b1), float(b2)), []).append(
            _ADAM.pack(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(),
                       float(group["lr"]), _advance(st["step"]), float(group["eps"])))
    _written(written)
    for (index, b1, b2), items in by_cfg.items():
        device = torch.device("cuda", index)
        with _capi.on(device):
            if norm is None:
                rc = lib.vr_adam_step(b"".join(items), len(items), b1, b2, -1.0, _capi.stream_of(device))
            else:
                rc = lib.vr_adam_step_clipped(b"".join(items), len(items), b1, b2, -1.0, norm.data_ptr(), max_grad_norm,
                                              _capi.stream_of(device))
        _capi.check(rc)
    return norm


def add_densification_stats(viewspace_point_grad, radii, xyz_gradient_accum, denom, max_radii2D):
    """In place, for every Gaussian with radii > 0 (the reference's visibility_filter, gaussian_renderer/__init__.py:117):
    xyz_gradient_accum += ||viewspace_point_grad[:, :2]||, denom += 1 (scene/gaussian_model.py:411-413) and
    max_radii2D = max(max_radii2D, radii) (train.py:299)."""
    P = radii.shape[0]
    for name, t, shape, dt in (("viewspace_point_grad", viewspace_point_grad, (P, 3), torch.float32),
                               ("radii", radii, (P,), torch.int32),
                               ("xyz_gradient_accum", xyz_gradient_accum, (P, 1), torch.float32),
                               ("denom", denom, (P, 1), torch.float32), ("max_radii2D", max_radii2D, (P,), torch.float32)):
        if not t.is_cuda:
            raise ValueError(f"{name} must be a GPU tensor (there is no CPU path)")
        if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dt} {shape} (got {t.dtype} {tuple(t.shape)})")
    lib = _capi.load()
    with torch.cuda.device(radii.device):
        rc = lib.vr_densify_stats(_capi.ptr(viewspace_point_grad), _capi.ptr(radii), P, _capi.ptr(xyz_gradient_accum),
                                  _capi.ptr(denom), _capi.ptr(max_radii2D),
                                  torch.cuda.current_stream(radii.device).cuda_stream)
    _capi.check(rc)


# ---------------------------------------------------------------------------------------------------------------------
# Densification (csrc/densify.hip).  The model's tensors are found the way the reference finds them: by the "name" of their
# optimizer group (scene/gaussian_model.py:159-166: xyz, f_dc, f_rest, opacity, scaling, rotation; one tensor per group).
DENSIFY_NAMES = ("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation")
_ROLES = {"xyz": 1, "scaling": 2}


def _named_groups(optimizer):
    groups = {}
    for group in optimizer.param_groups:
        if len(group["params"]) != 1:
            raise ValueError("densification expects one tensor per optimizer group (scene/gaussian_model.py:313)")
        groups[group.get("name")] = group
    missing = [n for n in DENSIFY_NAMES if n not in groups]
    if missing:
        raise ValueError(f"optimizer groups named {missing} are missing (scene/gaussian_model.py:159-166)")
    return groups


def _model_tensor(name, p, P, width=None):
    if not p.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (there is no CPU path)")
    if p.dtype != torch.float32 or p.dim() < 2 or p.shape[0] != P or not p.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 [{P}, ...] (got {p.dtype} {tuple(p.shape)})")
    if width is not None and math.prod(p.shape[1:]) != width:
        raise ValueError(f"{name} must have {width} values per Gaussian (got {tuple(p.shape)})")


def densify_and_prune(optimizer, xyz_gradient_accum, denom, max_grad, min_opacity, extent, max_screen_size,
                      percent_dense, noise=None, generator=None, empty_cache=True, prune=True):
    """GaussianModel.densify_and_prune (scene/gaussian_model.py:384-403) on the tensors of `optimizer`'s six named groups:
    clone the small Gaussians whose mean screen-space gradient `xyz_gradient_accum / denom` reaches `max_grad`, replace
    the large ones by two samples, prune by opacity (and, if `max_screen_size` is truthy, by world size -- the
    reference's screen-size test never fires, see include/vegs_optim.h), carrying the Adam moments of the survivors
    along and starting the new rows' at zero.  As in the reference the optimizer ends up with NEW nn.Parameter objects
    (state re-keyed, "step" untouched); they are returned as {name: parameter} like its `optimizable_tensors`, together
    with the fresh statistics (xyz_gradient_accum, denom, max_radii2D) = zeros of the new length (:349-351).

    One planned gather instead of the reference's two concatenations and two mask passes per tensor: the result has
    the same rows in the same order.  `noise` [2 S, 3] is the unit-normal draw behind torch.normal (:367), S = number
    of split Gaussians; drawn here with `generator` when not given -- pass it to make the step reproducible.
    `empty_cache`: finish with torch.cuda.empty_cache() as the reference does (:403).  `prune=False` is the reference's
    argument of that name (:384, :397): clone and split only, nothing is pruned by opacity or size."""
    groups = _named_groups(optimizer)
    par = {n: groups[n]["params"][0] for n in DENSIFY_NAMES}
    P = par["xyz"].shape[0]
    dev = par["xyz"].device
    for n, w in (("xyz", 3), ("opacity", 1), ("scaling", 3), ("rotation", 4), ("f_dc", None), ("f_rest", None)):
        _model_tensor(n, par[n], P, w)
    for n, t in (("xyz_gradient_accum", xyz_gradient_accum), ("denom", denom)):
        if not t.is_cuda or t.dtype != torch.float32 or t.numel() != P or not t.is_contiguous():
            raise ValueError(f"{n} must be a contiguous float32 GPU tensor with one value per Gaussian")
    lib = _capi.load()
    settings = _capi.VrDensifySettings(float(max_grad), float(min_opacity), float(extent), float(percent_dense),
                                       2 if not prune else (1 if max_screen_size else 0))
    stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev), torch.no_grad():
        plan = torch.empty(max(int(lib.vr_densify_plan_words(P)), 1), dtype=torch.int32, device=dev)
        counts = torch.empty(8, dtype=torch.int32, device=dev)
        _capi.check(lib.vr_densify_plan(_capi.ptr(par["opacity"]), _capi.ptr(par["scaling"]), _capi.ptr(xyz_gradient_accum),
                                        _capi.ptr(denom), P, C.byref(settings), plan.data_ptr(), counts.data_ptr(), stream))
        n_out, _, _, _, n_split = (int(c) for c in counts[:5].tolist())       # the one host round trip of the step
        if noise is None:
            noise = torch.randn((2 * n_split, 3), dtype=torch.float32, device=dev, generator=generator)
        if not noise.is_cuda or noise.dtype != torch.float32 or tuple(noise.shape) != (2 * n_split, 3):
            raise ValueError(f"noise must be a float32 GPU tensor [{2 * n_split}, 3] (two samples per split Gaussian)")
        noise = noise.contiguous()
        new, moments, items = {}, {}, []
        for n in DENSIFY_NAMES:
            p = par[n]
            st = optimizer.state.get(p, None)
            have = st is not None and "exp_avg" in st
            new[n] = torch.empty((n_out,) + tuple(p.shape[1:]), dtype=torch.float32, device=dev)
            m_src = v_src = m_dst = v_dst = None
            if have:
                m_src, v_src = st["exp_avg"], st["exp_avg_sq"]
                if m_src.shape != p.shape or v_src.shape != p.shape or not m_src.is_contiguous() or not v_src.is_contiguous():
                    raise ValueError(f"optimizer state of {n} does not match its parameter")
                m_dst, v_dst = torch.empty_like(new[n]), torch.empty_like(new[n])
                moments[n] = (m_dst, v_dst)
            if math.prod(p.shape[1:]) == 0:      # f_rest of a degree-0 model is [P,0,3]: nothing to move
                continue
            items.append(_capi.VrDensifyTensor(_capi.ptr(p), _capi.ptr(new[n]), _capi.ptr(m_src), _capi.ptr(m_dst),
                                               _capi.ptr(v_src), _capi.ptr(v_dst), math.prod(p.shape[1:]), _ROLES.get(n, 0)))
        if n_out > 0 and items:
            arr = (_capi.VrDensifyTensor * len(items))(*items)
            _capi.check(lib.vr_densify_apply(plan.data_ptr(), n_out, n_split, arr, len(items), _capi.ptr(par["scaling"]),
                                             _capi.ptr(par["rotation"]), _capi.ptr(noise), stream))
    out = {}
    for n in DENSIFY_NAMES:                      # _prune_optimizer / cat_tensors_to_optimizer's re-keying (:278-331)
        group, old = groups[n], par[n]
        stored = optimizer.state.get(old, None)
        param = torch.nn.Parameter(new[n].requires_grad_(True))
        if stored is not None:
            if n in moments:
                stored["exp_avg"], stored["exp_avg_sq"] = moments[n]
            del optimizer.state[old]
            optimizer.state[param] = stored
        group["params"][0] = param
        out[n] = param
    stats = (torch.zeros((n_out, 1), dtype=torch.float32, device=dev), torch.zeros((n_out, 1), dtype=torch.float32, device=dev),
             torch.zeros((n_out,), dtype=torch.float32, device=dev))
    if empty_cache:
        # as the reference does at the end of the step (:403): every per-Gaussian buffer changes size now, and the caching
        # allocator would otherwise keep the old generation's blocks (a 3000-iteration soak: 10 GB reserved for 0.6 GB in use)
        del new, moments, items, plan, counts, par
        torch.cuda.empty_cache()
    return out, stats


def reset_opacity(optimizer, cap=0.01):
    """GaussianModel.reset_opacity (scene/gaussian_model.py:215-218): opacity = inverse_sigmoid(min(sigmoid(opacity), 0.01))
    as a NEW nn.Parameter of the "opacity" group with zeroed Adam moments (replace_tensor_to_optimizer, :263-276); one
    launch.  Returns the parameter."""
    group = None
    for g in optimizer.param_groups:
        if g.get("name") == "opacity":
            group = g
    if group is None or len(group["params"]) != 1:
        raise ValueError('the optimizer has no single-tensor group named "opacity"')
    old = group["params"][0]
    if not old.is_cuda or old.dtype != torch.float32 or not old.is_contiguous():
        raise ValueError("opacity must be a contiguous float32 GPU tensor (there is no CPU path)")
    stored = optimizer.state.get(old, None)
    with torch.no_grad():
        new = old.detach().clone()
        m = v = None
        if stored is not None and "exp_avg" in stored:
            m, v = torch.empty_like(new), torch.empty_like(new)
        with torch.cuda.device(old.device):
            _capi.check(_capi.load().vr_reset_opacity(_capi.ptr(new), _capi.ptr(m), _capi.ptr(v), new.numel(), float(cap),
                                                      torch.cuda.current_stream(old.device).cuda_stream))
    param = torch.nn.Parameter(new.requires_grad_(True))
    if stored is not None:
        if m is not None:
            stored["exp_avg"], stored["exp_avg_sq"] = m, v
        del optimizer.state[old]
        optimizer.state[param] = stored
    group["params"][0] = param
    return param


# ---------------------------------------------------------------------------------------------------------------------
# Factored SH gradients.  The rasterizer can return, instead of dL/dshs [P,M,3], its rank-1 factor: the clamp-masked
# dL/d(colour) [P,3] of the view (GaussianRasterizer(..., sh_color_grad=sink)); dL/dshs[i,k,c] = basis_k(dir_i) *
# factor[i,c].  A view-sharded job all-gathers those 3 floats per Gaussian and view (vegs_amd.dist.exchange_factored)
# and every rank rebuilds -- or, better, consumes -- the sum over views locally.

def _check_factor_inputs(means3D, campos, factors):
    if not (means3D.is_cuda and campos.is_cuda and factors.is_cuda):
        raise ValueError("means3D, campos and factors must be GPU tensors (there is no CPU path)")
    P = means3D.shape[0]
    if means3D.dtype != torch.float32 or tuple(means3D.shape) != (P, 3):
        raise ValueError("means3D must be float32 [P,3]")
    if campos.dtype != torch.float32 or campos.dim() != 2 or campos.shape[1] != 3:
        raise ValueError("campos must be float32 [n_views,3]")
    n = campos.shape[0]
    if factors.dtype != torch.float32 or tuple(factors.shape) != (n, P, 3):
        raise ValueError(f"factors must be float32 [{n},{P},3] (got {tuple(factors.shape)})")
    # the P rows may be the HEAD of longer per-view blocks (the static model's rows of an all-gathered
    # [n_views, P + instance rows, 3]): passed with its view stride instead of a copy
    if not (factors.stride(2) == 1 and factors.stride(1) == 3 and (n == 1 or factors.stride(0) >= 3 * P)):
        factors = factors.contiguous()
    stride = factors.stride(0) if n > 1 else 0
    return P, n, means3D.contiguous(), campos.contiguous(), factors, stride


def sh_grad_from_factors(means3D, campos, factors, sh_degree, M, scale=1.0, split=False):
    """Dense dL/dshs from the factors of `n_views` views: scale * sum_v basis(dir(means3D, campos[v])) x factors[v].
    Returns [P,M,3], or (dc [P,1,3], rest [P,M-1,3]) with split=True (the model's own storage)."""
    P, n, means3D, campos, factors, fstride = _check_factor_inputs(means3D, campos, factors)
    dev = means3D.device
    if split:
        out = torch.empty((P, 1, 3), dtype=torch.float32, device=dev)
        rest = torch.empty((P, M - 1, 3), dtype=torch.float32, device=dev)
    else:
        out, rest = torch.empty((P, M, 3), dtype=torch.float32, device=dev), None
    with torch.cuda.device(dev):
        rc = _capi.load().vr_sh_grad_from_factors(_capi.ptr(means3D), P, _capi.ptr(campos), _capi.ptr(factors), n, fstride,
                                                  int(sh_degree), int(M), float(scale), _capi.ptr(out), _capi.ptr(rest),
                                                  torch.cuda.current_stream(dev).cuda_stream)
    _capi.check(rc)
    return (out, rest) if split else out


def _sh_state(opt, p):
    for group in opt.param_groups:
        for q in group["params"]:
            if q is p:
                st = opt.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                # the same checks torch.optim.Adam's step makes: densification code replaces these tensors in place
                # (scene/gaussian_model.py:263-331) and a mismatch would be written out of bounds by the kernel
                for name in ("exp_avg", "exp_avg_sq"):
                    t = st[name]
                    if t.shape != p.shape or t.dtype != torch.float32 or not t.is_cuda or t.device != p.device \
                            or not t.is_contiguous():
                        raise ValueError(f"optimizer state {name} must be a contiguous float32 tensor shaped like its "
                                         f"parameter {tuple(p.shape)} on {p.device} (got {tuple(t.shape)}, {t.dtype}, {t.device})")
                return group, st
    raise ValueError("parameter is not in the optimizer")


@torch.no_grad()
def adam_step_sh_factored(opt, features_dc, features_rest, means3D, campos, factors, sh_degree, scale=1.0,
                          max_grad_norm=None, grad_norm=None):
    """One Adam step of the SH parameters (features_dc [P,1,3] + features_rest [P,M-1,3], or the whole [P,M,3] tensor with
    features_rest=None) of optimizer `opt` (vegs_amd.optim.Adam or torch.optim.Adam: same state layout) straight from
    the factors -- the dense gradient is built per Gaussian in registers and never written.  Equivalent to setting
    .grad = sh_grad_from_factors(...) on the two parameters and stepping only them.

    max_grad_norm: clip this gradient as step_many does.  grad_norm: the joint norm (optim.grad_norm with this gradient among
    its sh_factors); without it the norm is this gradient's own.  Returns the norm then."""
    if max_grad_norm is None:
        if grad_norm is not None:
            raise ValueError("grad_norm without max_grad_norm")
    else:
        max_grad_norm = _check_max_norm(max_grad_norm)
    P, n, means3D, campos, factors, fstride = _check_factor_inputs(means3D, campos, factors)
    M = features_dc.shape[1] + (features_rest.shape[1] if features_rest is not None else 0)
    items, states, written, betas, eps = [], [], [], None, None
    for p in (features_dc, features_rest):
        if p is None:
            items.append(None)
            continue
        if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
            raise ValueError("SH parameters must be contiguous float32 GPU tensors")
        group, st = _sh_state(opt, p)
        if betas is None:
            betas, eps = tuple(group["betas"]), float(group["eps"])
        elif betas != tuple(group["betas"]) or eps != float(group["eps"]):
            raise ValueError("features_dc and features_rest must share betas and eps")
        items.append(_capi.VrShAdamTensor(p.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(),
                                          float(group["lr"]), int(st["step"].item()) + 1))
        states.append(st)
        written += (p, st["exp_avg"], st["exp_avg_sq"])
    K = (int(sh_degree) + 1) ** 2
    if not 0 <= int(sh_degree) <= 3 or M < K:
        raise ValueError(f"sh_degree {sh_degree} needs {K} coefficients, the parameters hold {M}")
    dev = means3D.device
    norm = None
    if max_grad_norm is not None:
        if grad_norm is not None:
            _check_norm(grad_norm, dev)
        norm = grad_norm if grad_norm is not None else _norm_of({}, 2, [(means3D, campos, factors, sh_degree, scale)])
    args = (_capi.ptr(means3D), P, _capi.ptr(campos), _capi.ptr(factors), n, fstride, int(sh_degree), int(M), float(scale),
            C.byref(items[0]), C.byref(items[1]) if items[1] is not None else None, betas[0], betas[1], eps)
    _written(written)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        if norm is None:
            rc = _capi.load().vr_sh_adam_step(*args, stream)
        else:
            rc = _capi.load().vr_sh_adam_step_clipped(*args, norm.data_ptr(), max_grad_norm, stream)
    _capi.check(rc)
    for st in states:          # the step counters advance only once every check and the call itself have passed
        st["step"] += 1
    return norm
