"""Optimiser of force-loss training: :class:`AdamW` over all of a model's tensors in a few launches, with its
moments in 32 or 8 bits, and :func:`grad_norm`, the global gradient norm that clips its step.

Nothing here reads the device: the clipping factor, the step counts and the decision to leave out a step whose
gradients are not finite stay in device memory (the reference's trainer reads a flag back for the latter,
pipeline/trainer.py:397-414), so a training step can be captured in a CUDA graph.
"""
from __future__ import annotations

from array import array
from contextlib import nullcontext
from operator import attrgetter, is_

import torch

from . import _lib
from ._lib import check, ptr, require_cuda, stream_of

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 256          # elements that share a scale; every tensor's state starts at a multiple


_dtype = attrgetter("dtype")


def _address(a):
    return a.buffer_info()[0]


def _pointers(tensors):
    return array("Q", map(torch.Tensor.data_ptr, tensors))


def _zeros(typecode, n):
    return array(typecode, (0,)) * n


def _table(tensors):
    """``(addresses, sizes, type code, device index)`` of a list of tensors in one call, or None where they are
    not all alike (see ``csrc/e2a_torch.cpp``)."""
    n = len(tensors)
    at, numel, two = _zeros("Q", n), _zeros("q", n), _zeros("i", 2)
    if _lib.load_torch().e2a_tensor_table(tensors, n, _address(at), _address(numel), _address(two), _address(two) + 4):
        return None
    return at, numel, two[0], two[1]


def _one_device(tensors, what):
    devices = set(map(torch.Tensor.get_device, tensors))
    if len(devices) > 1 or min(devices) < 0:
        require_cuda(*tensors)
        raise ValueError(f"{what} are on more than one device")
    return tensors[0].device


def _contiguous(tensors):
    if any(t.layout != torch.strided for t in tensors):
        raise TypeError("expected strided tensors")
    return [t.detach().contiguous() for t in tensors]


def _gradients(params):
    """The parameters' gradients, contiguous.  A gradient can differ from its parameter in type (``grad_dtype``) or,
    after ``p.data = ...``, in size and device; the kernels read both alike."""
    for p in params:
        if p.grad.dtype != p.dtype:
            raise TypeError(f"a {p.dtype} parameter has a {p.grad.dtype} gradient")
        if p.grad.numel() != p.numel() or p.grad.device != p.device:
            raise ValueError(f"a parameter of {p.numel()} values on {p.device} has a gradient of {p.grad.numel()} on "
                             f"{p.grad.device}")
    return _contiguous([p.grad for p in params])


def _by_type(what, tensors, *others):
    """``[(type code, tensors, *others)]``: the lists split by the tensors' types."""
    kinds = set(map(_dtype, tensors))
    if not kinds <= _DTYPES.keys():
        raise TypeError(f"{what} takes float32, bfloat16 or float16 tensors, got {kinds - _DTYPES.keys()}")
    keep = {d: [k for k, t in enumerate(tensors) if t.dtype == d] for d in _DTYPES if d in kinds}
    return [(_DTYPES[d], *([x[k] for k in ks] for x in (tensors, *others))) for d, ks in keep.items()]


def _norm(dev, lists):
    """The norm of ``lists`` = [(type code, number, where the tensors' addresses and sizes stand)] of contiguous tensors
    on the current device."""
    lib, stream = _lib.load(), stream_of(dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = sum(lib.e2a_grad_norm_workspace_bytes(n) for _, n, _, _ in lists)
    ws = torch.empty(max(size, 8), dtype=torch.uint8, device=dev)
    base = ws.data_ptr()
    if len(lists) == 1:
        (code, n, at, numel), = lists
        check(lib.e2a_grad_norm(at, numel, n, code, base, size, norm.data_ptr(), stream),
              "e2a_grad_norm")
        return norm
    done, count = 0, array("q", (0,))
    for code, n, at, numel in lists:
        check(lib.e2a_sum_squares(at, numel, n, code, base + 8 * done, size - 8 * done,
                                  _address(count), stream), "e2a_sum_squares")
        done += count[0]
    check(lib.e2a_norm_of_squares(base, done, norm.data_ptr(), stream), "e2a_norm_of_squares")
    return norm


def grad_norm(tensors):
    """The global L2 norm ``sqrt(sum of all squares)`` of ``tensors`` (float32, bfloat16 or float16 on one CUDA
    device, any shapes) as a 0-dim float32 tensor there: sums in 64 bits, in a fixed order, no host read.  An
    empty list has norm 0 on the current device."""
    tensors = list(tensors)
    found = _table(tensors) if tensors else None
    if found is not None:
        at, numel, code, index = found
        dev, tables = torch.device("cuda", index), [(code, len(at), at, numel)]
    else:
        dev = _one_device(tensors, "the tensors") if tensors else torch.device("cuda", torch.cuda.current_device())
        tensors = _contiguous(tensors)
        tables = [(code, len(ts), _pointers(ts), array("q", map(torch.Tensor.numel, ts)))
                  for code, ts in _by_type("grad_norm", tensors)]
    with torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else nullcontext():
        return _norm(dev, [(code, n, _address(at), _address(numel)) for code, n, at, numel in tables])


def _rate(lr, device):
    """``(value, device address or None)`` of a group's learning rate."""
    if not isinstance(lr, torch.Tensor) or not lr.is_cuda:
        return float(lr), None
    if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != device:
        raise ValueError("a tensor lr must be one float32 value on the parameters' device")
    return 0.0, lr.data_ptr()


class _Flat:
    """The state of one parameter group: flat moments, every tensor at a multiple of 256 elements, and a step
    count per tensor."""

    def __init__(self, params, bits):
        self.device, self.params = _one_device(params, "a group's parameters"), list(params)
        self.numel, self.offset, end = array("q", map(torch.Tensor.numel, params)), array("q"), 0
        for n in self.numel:
            self.offset.append(end)
            end += -(-n // BLOCK) * BLOCK
        self.slot = array("i", range(len(params)))
        self.at = _address(self.numel), _address(self.offset)
        self.elements, self.bits = end, bits
        kind = torch.float32 if bits == 32 else torch.uint8
        self.buffers = {"step": torch.zeros(len(params), dtype=torch.int32, device=self.device),
                        "exp_avg": torch.zeros(end, dtype=kind, device=self.device),
                        "exp_avg_sq": torch.zeros(end, dtype=kind, device=self.device)}
        if bits == 8:
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                self.buffers[k] = torch.zeros(end // BLOCK, dtype=torch.uint8, device=self.device)
        self.entries = [self.view(i, p) for i, p in enumerate(self.params)]
        self.values = [tuple(e.values()) for e in self.entries]
        self.names = tuple(self.entries[0]) if self.entries else ()
        self.filled = self.stale = False

    def view(self, i, param):
        """The state of tensor ``i``: views of the flat buffers."""
        n, o = self.numel[i], self.offset[i]
        out = {"step": self.buffers["step"][i], "exp_avg": self.buffers["exp_avg"][o:o + n].view(param.shape),
               "exp_avg_sq": self.buffers["exp_avg_sq"][o:o + n].view(param.shape)}
        for k in ("exp_avg_scale", "exp_avg_sq_scale"):
            if k in self.buffers:
                out[k] = self.buffers[k][o // BLOCK:(o + n + BLOCK - 1) // BLOCK]
        return out

    def belongs_to(self, params):
        return len(params) == len(self.params) and all(map(is_, params, self.params))

    def fits(self, params):
        return self.belongs_to(params) and all(p.numel() == n and p.device == self.device
                                               for p, n in zip(params, self.numel))

    def held_in(self, state):
        """Whether an optimiser's ``state`` has this state's views, and nothing else, for its parameters."""
        return all(state.get(p) is e and len(e) == len(v) and all(map(is_, e.values(), v))
                   for p, e, v in zip(self.params, self.entries, self.values))

    def fill(self, given):
        """Takes the states ``given`` for its tensors, where None zeros; what are its own views already stays.  Nothing
        is changed where one does not fit."""
        names = self.names
        for p, e, v in zip(self.params, given, self.values):
            if e is not None and (set(e) != set(names) or any(
                    e[k].shape != t.shape or (e[k].dtype != t.dtype and k != "step") for k, t in zip(names, v))):
                raise ValueError(f"the state of a parameter of shape {list(p.shape)} is not one of {self.bits}-bit moments")
        # copies first: a given tensor can be a view of another's place
        moved = [(t, e[k].clone()) for e, v in zip(given, self.values) if e is not None
                 for k, t in zip(names, v) if e[k] is not t]
        if self.filled:
            zeros = self.buffers.values() if not any(given) else [t for e, v in zip(given, self.values) if e is None
                                                                  for t in v]
            for t in zeros:
                t.zero_()
        for t, value in moved:
            t.copy_(value)
        self.entries = [dict(zip(names, v)) for v in self.values]
        self.filled, self.stale = True, False


# group options that change PyTorch's AdamW or this one's arguments, with the only value that they may have here
_FIXED = {"maximize": False, "amsgrad": False, "differentiable": False, "decoupled_weight_decay": True,
          "state_bits": None, "max_grad_norm": None}


def _check_options(group):
    for k, only in _FIXED.items():
        if k in group and (only is None or bool(group[k]) != only):
            raise ValueError(f"AdamW takes no {k}={group[k]!r} for a group")


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with PyTorch's arguments and update; parameters in float32, bfloat16 or
    float16, contiguous, the arithmetic in fp32 with one rounding to the parameter's type; ``eps`` is 0 or at least
    2^-126.

    * ``state_bits``: 32 = fp32 moments; 8 = one byte per element and moment plus one scale byte per 256
      (see ``csrc/e2a_optim.cu``).  An 8-bit value is rounded either way as often as it is near, but what passes a
      block's largest code stays there: random gradients leave sqrt(v) 1.4% low in the mean and the largest of each
      256 about 40%, gradients that never change leave it at 1/8 to 1/4 of its value (steps up to 8 times as long).
    * ``max_grad_norm``: clip the gradients of each step to this global norm (over all groups) inside the update;
      the gradients themselves are left as they are.  The norm of the last step is ``last_grad_norm`` (0-dim
      tensor on the device).  A step whose norm is not finite changes nothing, step counts included.
    * ``lr`` of a group: a float, or a float32 tensor of one element on the parameters' device, which a captured
      step reads anew at every replay.

    A group's options that would change the update and that there are none of here (``maximize``, ``amsgrad``,
    ``differentiable``, ``decoupled_weight_decay=False``) are refused, in a loaded state too.

    Parameters without a gradient are left out of a step, each has its own step count.  State entries
    (``step``, ``exp_avg``, ``exp_avg_sq`` and, in 8 bits, their ``_scale``) are views of one flat buffer per
    group (:meth:`flat_state`); ``state_dict`` / ``load_state_dict`` keep types and bits.  As with PyTorch's, the
    state belongs to the parameter: one that replaces another, or whose entry in ``state`` was cleared, starts anew,
    and groups may be reordered, shortened or removed between steps (the next step then lays their state out again, in
    the same memory while a group's parameters are the same, so that a captured step goes on from there)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 max_grad_norm=None):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits={state_bits!r}: expected 32 or 8")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm={max_grad_norm!r} must be positive")
        self.state_bits, self.max_grad_norm, self.last_grad_norm = state_bits, max_grad_norm, None
        self._flat, self._held = {}, []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            _check_options(g)
            b1, b2 = g["betas"]
            if not (0 <= b1 < 1 and 0 <= b2 < 1 and g["eps"] >= 0 and g["weight_decay"] >= 0):
                raise ValueError(f"invalid betas {g['betas']}, eps {g['eps']} or weight_decay {g['weight_decay']}")
            if 0 < g["eps"] < 2.0 ** -126:
                raise ValueError(f"eps={g['eps']} is below the normal fp32 range: 0, or at least 2^-126")
            if not isinstance(g["lr"], torch.Tensor) and not g["lr"] >= 0:
                raise ValueError(f"invalid lr {g['lr']}")
            if len(set(map(id, g["params"]))) != len(g["params"]):
                raise ValueError("a parameter appears twice in a group")
        except ValueError:
            self.param_groups.pop()
            raise

    # -- state -------------------------------------------------------------------------------------
    def _sync(self):
        """Marks the layouts that ``state`` no longer is the views of, whoever changed it; what it holds is laid out again
        where a group needs it."""
        if _lib.load_torch().e2a_state_is_held(self.state, self._held, len(self._held)):
            self._flat = {i: f for i, f in self._flat.items() if i < len(self.param_groups)}
            for f in self._flat.values():
                f.stale = f.stale or not f.held_in(self.state)
            self._hold()

    def _hold(self):
        """Notes ``state`` as it is: its keys, entries and their values."""
        self._held = [x for p, e in self.state.items()
                      for x in (p, e, tuple(e.values()) if isinstance(e, dict) else ())]

    def _group_state(self, i):
        self._sync()
        flat, params = self._flat.get(i), self.param_groups[i]["params"]
        return flat if flat is not None and not flat.stale and flat.belongs_to(params) else self._lay_out(i)

    def _lay_out(self, i):
        """A flat state for group ``i``, with what ``state`` has for its parameters and zeros for the others; in the
        memory of the one that it has where the parameters are the same, so that captured steps stay good."""
        params = self.param_groups[i]["params"]
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW's state would be made inside a graph capture, and made anew by every replay: call "
                               "flat_state() for each group before it")
        flat = self._flat.get(i)
        if flat is None or not flat.fits(params):
            flat = _Flat(params, self.state_bits)
        with torch.no_grad():
            flat.fill([self.state.get(p) or None for p in params])
        self.state.update(zip(params, flat.entries))
        self._flat[i] = flat
        self._hold()
        return flat

    def flat_state(self, group=0):
        """The flat buffers of a group: ``step`` [tensors], ``exp_avg`` and ``exp_avg_sq`` [elements] (each tensor
        from the next multiple of 256 on), in 8 bits also ``exp_avg_scale`` / ``exp_avg_sq_scale``."""
        return dict(self._group_state(group).buffers)

    def moments(self, group=0):
        """``(exp_avg, exp_avg_sq)`` of a group as flat fp32 values (the buffers themselves with 32 bits)."""
        flat = self._group_state(group)
        b = flat.buffers
        if flat.bits == 32:
            return b["exp_avg"], b["exp_avg_sq"]
        with torch.cuda.device(flat.device):
            m = torch.empty(flat.elements, dtype=torch.float32, device=flat.device)
            v = torch.empty_like(m)
            check(_lib.load().e2a_moments_unpack(ptr(b["exp_avg"]), ptr(b["exp_avg_sq"]), ptr(b["exp_avg_scale"]),
                                                 ptr(b["exp_avg_sq_scale"]), flat.elements, ptr(m), ptr(v),
                                                 stream_of(flat.device)), "e2a_moments_unpack")
        return m, v

    def load_state_dict(self, state_dict):
        """Restores types and bits as they were saved; a state of other bits or shapes is refused."""
        groups = state_dict["param_groups"]
        held = state_dict["state"]
        for g in groups:
            _check_options(g)
        wanted = {"step", "exp_avg", "exp_avg_sq"} | (
            {"exp_avg_scale", "exp_avg_sq_scale"} if self.state_bits == 8 else set())
        kind = torch.float32 if self.state_bits == 32 else torch.uint8
        for k, s in held.items():
            if set(s) != wanted or s["exp_avg"].dtype != kind or s["exp_avg_sq"].dtype != kind:
                raise ValueError(f"state of parameter {k} is not one of {self.state_bits}-bit moments")
        pairs = [(i, p) for g, mine in zip(groups, self.param_groups) for i, p in zip(g["params"], mine["params"])]
        for i, p in pairs:
            scales = (-(-p.numel() // BLOCK),)
            shapes = {"step": (), "exp_avg": p.shape, "exp_avg_sq": p.shape, "exp_avg_scale": scales,
                      "exp_avg_sq_scale": scales}
            if i in held and any(t.shape != shapes[k] for k, t in held[i].items()):
                raise ValueError(f"state of parameter {i} has another shape than the parameter's")
        flats = self._flat
        super().load_state_dict({"state": {}, "param_groups": groups})    # checks and takes the groups
        self._flat = flats
        for f in flats.values():
            f.stale = True
        for gi, (g, mine) in enumerate(zip(groups, self.param_groups)):
            if any(i in held for i in g["params"]):
                self.state.update((p, held[i]) for i, p in zip(g["params"], mine["params"]) if i in held)
                self._lay_out(gi)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_grad_norm": self.max_grad_norm,
                "last_grad_norm": self.last_grad_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._flat, self._held = {}, []
        for gi, g in enumerate(self.param_groups):      # a copy's state becomes views of its own flat buffers
            if any(self.state.get(p) for p in g["params"]):
                self._lay_out(gi)

    # -- the step ----------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._sync()
        work, keep = [], []
        for gi, g in enumerate(self.param_groups):
            work += self._group_work(gi, g, keep)
        if not work:
            return loss
        norm = None
        if self.max_grad_norm is not None:
            dev = work[0][1].device
            if any(w[1].device != dev for w in work):
                raise ValueError("the parameters to clip together are on more than one device")
            with torch.cuda.device(dev):
                norm = self.last_grad_norm = _norm(dev, [(w[3], w[4], w[6], w[7]) for w in work])
        for w in work:
            if w[1].device.index == torch.cuda.current_device():
                self._launch(*w, norm)
            else:
                with torch.cuda.device(w[1].device):
                    self._launch(*w, norm)
        return loss

    def _group_work(self, gi, group, keep):
        """The launches of a group: ``[(group, flat state, learning rate, type code, number of tensors, and where the
        addresses of the parameters and of their gradients, their sizes, state offsets and slots stand)]``; ``keep``
        holds what has to live until then."""
        _check_options(group)
        params = group["params"]
        if not params:
            return []
        flat = self._flat.get(gi)
        if flat is None or flat.stale:
            if all(p.grad is None for p in params):
                return []
            flat = self._lay_out(gi)
        rate = _rate(group["lr"], flat.device)
        found = self._read(group, flat, rate, keep)
        if found is None and not flat.belongs_to(params):
            flat = self._lay_out(gi)
            found = self._read(group, flat, rate, keep)
        if found is not None:
            return found
        index = [k for k, p in enumerate(params) if p.grad is not None]
        if not index:
            return []
        params = [params[k] for k in index]
        if _one_device(params, "a group's parameters") != flat.device:
            raise ValueError("the parameters have moved to another device than their state")
        if not all(map(torch.Tensor.is_contiguous, params)):
            raise ValueError("AdamW takes contiguous parameters")
        if any(p.numel() != flat.numel[k] for k, p in zip(index, params)):
            raise ValueError("a parameter has changed its size since its state was made")
        grads = _gradients(params)
        work = []
        for code, ps, gs, ks in _by_type("AdamW", params, grads, index):
            table = [_pointers(ps), _pointers(gs), *(array(a.typecode, [a[k] for k in ks])
                                                     for a in (flat.numel, flat.offset, flat.slot))]
            keep.append((grads, table))
            work.append((group, flat, rate, code, len(ps), *map(_address, table)))
        # the kernels write behind autograd's back: saved tensors and caches keyed on versions have to see it
        torch.autograd.graph.increment_version(params)
        return work

    @staticmethod
    def _read(group, flat, rate, keep):
        """The launch of a group whose parameters are those of ``flat`` and all alike, in one call; else None."""
        params, n = group["params"], len(flat.params)
        table = _zeros("q", 5 * n + 2)
        at = _address(table)
        if len(params) != n or _lib.load_torch().e2a_step_table(params, flat.params, n, flat.at[0], flat.at[1], at):
            return None
        two, count = divmod(table[5 * n], 1 << 32), table[5 * n + 1]
        if count == 0:
            return []
        if two[1] != flat.device.index:
            raise ValueError("the parameters have moved to another device than their state")
        keep.append(table)
        return [(group, flat, rate, two[0], count, at, at + 8 * n, at + 16 * n, at + 24 * n, at + 32 * n)]

    def _launch(self, group, flat, rate, code, count, at, grads, numel, offset, slot, norm):
        (beta1, beta2), b = group["betas"], flat.buffers
        m, v, ms, vs, step = (b[k].data_ptr() if k in b else None for k in (
            "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"))
        lib = _lib.load()
        ws = torch.empty(lib.e2a_adamw_workspace_bytes(count), dtype=torch.uint8, device=flat.device)
        check(lib.e2a_adamw_step(
            at, grads, numel, offset, slot, count, code, flat.bits, m, v, ms, vs, flat.elements, step, *rate, beta1,
            beta2, group["eps"], group["weight_decay"],
            None if norm is None else norm.data_ptr(), self.max_grad_norm or 0.0, ws.data_ptr(), ws.numel(),
            stream_of(flat.device)), "e2a_adamw_step")
