"""AdamW over many tensors at once, its moments held in 32 bits or in 8 (pin_adamw_step).

The optimiser beside the mapping loop's own Adam launches, for what a program trains through
autograd: heads, features and networks of any number of tensors in f32, f16 or bf16
(utils/tools.py:89-116 builds the reference's torch.optim.Adam from the same kinds of groups, and
its rates are the defaults here).  A step is one launch for up to 112 tensors of one group, type
and step count.

The state of a parameter group lies in flat arrays in which every parameter begins at a multiple
of 256 elements (``offsets``); ``state[p]`` holds views of them.  With state_bits 8 a moment takes
one byte per element and two bytes per 256, rounded so that its expectation is kept
(csrc/pin_adamw.hip).
"""
from array import array

import torch

from . import _lib

_SALT_SEED, _SALT_GROUP = 0x9E3779B1, 0xBB67AE85
_INF = float("inf")
_RATES = ("lr", "betas", "eps", "weight_decay", "state_bits", "master_weights")
_STATE_KEYS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_sq", "exponents")}


def _blocks(n):
    return -(-n // _lib.ADAMW_BLOCK)


def _has_master(group):
    return group["master_weights"] and any(p.dtype != torch.float32 for p in group["params"])


class _Arena:
    """The state of one parameter group."""

    def __init__(self, group, capturable):
        params = group["params"]
        bits = group["state_bits"]
        dev = params[0].device
        self.bits, self.device = bits, dev
        self.sizes = [p.numel() for p in params]
        self.offsets, total = [], 0
        for n in self.sizes:
            self.offsets.append(total)
            total += _blocks(n) * _lib.ADAMW_BLOCK
        self.total = total
        kind = torch.float32 if bits == 32 else torch.uint8
        self.m = torch.zeros((total,), dtype=kind, device=dev)
        self.v = torch.zeros((total,), dtype=kind, device=dev)
        self.exps = torch.zeros((total // _lib.ADAMW_BLOCK, 2), dtype=torch.int16, device=dev) if bits == 8 else None
        self.master = torch.zeros((total,), dtype=torch.float32, device=dev) if _has_master(group) else None
        self.master_weights = group["master_weights"]
        self.held = None
        self.index = dev.index
        self.c_sizes, self.c_offsets = array("q", self.sizes), array("q", self.offsets)
        # a step that a graph may replay counts on the device, all of the group's parameters together
        self.step_dev = torch.zeros((1,), dtype=torch.int64, device=dev) if capturable else None
        self.scalars = torch.zeros((_lib.ADAMW_SCALARS_BYTES,), dtype=torch.uint8, device=dev) if capturable else None
        self.start(params)
        self.written = self.arrays()      # by every step

    def arrays(self):
        return [x for x in (self.m, self.v, self.exps, self.master, self.step_dev) if x is not None]

    def start(self, params):
        """As before the first step, where it lies (a captured graph goes on with it)."""
        for x in self.arrays():
            x.zero_()
        if self.master is not None:
            for p, a, n in zip(params, self.offsets, self.sizes):
                self.master[a:a + n] = p.detach().reshape(-1)
        self.wide = [p.dtype == torch.float32 for p in params]
        self.steps = [0] * len(params)
        self.together = True              # all of them are the same

    def fits(self, group):
        return (self.sizes == [p.numel() for p in group["params"]] and (self.master is not None) == _has_master(group)
                and all(p.device == self.device for p in group["params"]))

    def views(self, i, shape):
        """The parameter's part of each array."""
        a, n = self.offsets[i], self.sizes[i]
        one = {"exp_avg": self.m[a:a + n].view(shape), "exp_avg_sq": self.v[a:a + n].view(shape)}
        if self.exps is not None:
            one["exponents"] = self.exps[a // _lib.ADAMW_BLOCK:a // _lib.ADAMW_BLOCK + _blocks(n)]
        if self.master is not None:
            one["master"] = self.master[a:a + n].view(shape)
        return one


class AdamW(torch.optim.Optimizer):
    """Parameters p with gradients g, per step t of the parameter:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    lr, betas, eps, weight_decay, state_bits (32 or 8) and master_weights (16-bit parameters keep a
    copy in 32 bits that the steps go on from) may differ by parameter group; parameters of a group
    share a device and are contiguous.  seed chooses the 8-bit moments' rounding.

    capturable: step() may be captured into a graph after one eager step; a group's parameters then
    all have gradients and count steps together, and lr may be a float32 tensor on the device that
    replays read (a number is taken as it was when captured).  A replay cannot mark the parameters as
    modified: what is derived from them (a map's or decoder's views among it) goes by
    torch.autograd.graph.increment_version(parameters) after it.

    The state is made at the first step (or by load_state_dict); parameters are neither added to a
    group, reshaped nor moved to another device afterwards."""

    def __init__(self, params, lr=0.01, betas=(0.9, 0.99), eps=1e-15, weight_decay=0.0, *, state_bits=32,
                 master_weights=False, capturable=False, seed=0):
        self.capturable, self.seed = bool(capturable), int(seed)
        self._arenas = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=bool(master_weights)))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def __getstate__(self):
        return {**super().__getstate__(), "capturable": self.capturable, "seed": self.seed, "_arenas": self._arenas}

    def _check_lr(self, lr, device):
        if not self.capturable or lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != device:
            raise ValueError("AdamW: a tensor lr must be one float32 on the parameters' device, with capturable=True")

    @staticmethod
    def _check_rates(group, lr):
        b1, b2 = group["betas"]
        if (0.0 <= lr < _INF and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and 0.0 <= group["eps"] < _INF
                and 0.0 <= group["weight_decay"] < _INF and group["state_bits"] in _STATE_KEYS):
            return
        if not 0.0 <= lr < _INF:
            raise ValueError(f"AdamW: lr must be >= 0 (got {lr})")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1) (got {group['betas']})")
        if group["state_bits"] not in _STATE_KEYS:
            raise ValueError(f"AdamW: state_bits must be 32 or 8 (got {group['state_bits']})")
        raise ValueError(f"AdamW: eps and weight_decay must be >= 0 (got {group['eps']}, {group['weight_decay']})")

    def _check_group(self, group):
        params = group["params"]
        if isinstance(group["lr"], torch.Tensor):
            self._check_lr(group["lr"], params[0].device)
        self._check_rates(group, 0.0 if isinstance(group["lr"], torch.Tensor) else group["lr"])
        spans = []
        for p in params:
            if p.dtype not in _lib.TYPES:
                raise ValueError(f"AdamW: parameters must be float32, float16 or bfloat16 (got {p.dtype})")
            if p.layout != torch.strided or not p.is_contiguous():
                raise ValueError("AdamW: parameters must be contiguous")
            if p.device != params[0].device:
                raise ValueError("AdamW: the parameters of a group must be on one device")
            spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        for other in self.param_groups:
            if other is not group:
                spans += [(p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in other["params"]]
        spans = sorted(s for s in spans if s[1] > s[0])
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")

    def _show(self, arena, group):
        for i, p in enumerate(group["params"]):
            self.state[p] = arena.views(i, p.shape)

    def _arena(self, gi):
        group = self.param_groups[gi]
        gi %= len(self.param_groups)   # (the last group is also number -1)
        arena = self._arenas.get(gi)
        if arena is None:
            for p in group["params"]:
                _lib.require_device(p)
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: run one step before capturing one (it makes the state)")
            arena = self._arenas[gi] = _Arena(group, self.capturable)
            self._show(arena, group)
        elif group["params"] and group["params"][0] not in self.state:   # state was emptied: torch's optimisers begin anew
            if not arena.fits(group) or any(p in self.state for p in group["params"]):
                raise RuntimeError("AdamW: parameters were added to or taken from a group after its first step")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: run one step before capturing one (it makes the state)")
            arena.start(group["params"])
            self._show(arena, group)
        if len(arena.sizes) != len(group["params"]):
            raise RuntimeError("AdamW: parameters were added to or taken from a group after its first step")
        return arena

    def _check(self, arena, i, p, g):
        """One parameter and its gradient; the gradient as the kernel takes it."""
        if g.layout != torch.strided:
            raise RuntimeError("AdamW: sparse gradients are not implemented")
        if p.numel() != arena.sizes[i] or p.device != arena.device or not p.is_contiguous():
            raise RuntimeError("AdamW: a parameter was reshaped or moved after its first step")
        if g.dtype != p.dtype or g.device != arena.device or p.dtype not in _lib.TYPES or g.numel() != arena.sizes[i]:
            raise RuntimeError(f"AdamW: a {p.dtype} parameter on {p.device} has a {g.dtype} gradient on {g.device}")
        if arena.master_weights and (p.dtype == torch.float32) != arena.wide[i]:   # its copy is another's, or there is none
            raise RuntimeError(f"AdamW: a parameter with a copy in 32 bits became {p.dtype} after its first step")
        if p.is_neg():
            raise RuntimeError("AdamW: a parameter is a negated view")
        return g.resolve_neg().contiguous()

    def _gather(self, arena, group):
        """What has a gradient, checked: launches of (indexes or None for all, their type, addresses of the parameters and
        of the gradients)."""
        params = group["params"]
        n = len(params)
        if arena.together:   # the usual step: every parameter and every gradient as the kernel takes them
            ps, gs = array("Q", bytes(8 * n)), array("Q", bytes(8 * n))
            if _lib.torch_fn("pin_torch_gather")(params, n, arena.c_sizes.buffer_info()[0], arena.index, ps.buffer_info()[0],
                                   gs.buffer_info()[0]) >= 0 and not (
                    arena.master_weights and (params[0].dtype == torch.float32) != arena.wide[0]):
                return [(None, params[0].dtype, ps, gs)]
        grads = [p.grad for p in params]
        which = [i for i, g in enumerate(grads) if g is not None]
        if self.capturable and len(which) < n:
            raise RuntimeError("AdamW: with capturable=True every parameter of a group needs a gradient")
        some = {}
        held = arena.held = []   # copies made here live until the step is on its way
        for i in which:
            g = self._check(arena, i, params[i], grads[i])
            idx, ps, gs = some.setdefault((params[i].dtype, arena.steps[i]), ([], array("Q"), array("Q")))
            idx.append(i)
            ps.append(params[i].data_ptr())
            gs.append(g.data_ptr())
            held.append(g)
        return [(idx, dtype, ps, gs) for (dtype, _), (idx, ps, gs) in some.items()]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # everything is checked before anything is stepped, and the groups before any state is made
        groups, work = [], []
        for gi, group in enumerate(self.param_groups):
            params = group["params"]
            if not params or not (self.capturable or params[0].grad is not None or any(p.grad is not None for p in params)):
                continue
            _lib.require_device(params[0])
            if not self.capturable and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: capturing a step needs capturable=True (the step count is on the host)")
            lr = group["lr"]
            if isinstance(lr, torch.Tensor):
                self._check_lr(lr, params[0].device)
                lr = 0.0
            self._check_rates(group, lr)
            arena = self._arenas.get(gi)
            if arena is not None and (arena.bits != group["state_bits"] or (
                    arena.master_weights != group["master_weights"] and (arena.master is not None) != _has_master(group))):
                raise RuntimeError("AdamW: state_bits or master_weights changed after a group's first step")
            groups.append((gi, group))
        for gi, group in groups:
            arena = self._arena(gi)
            work.append((gi, group, arena, self._gather(arena, group)))
        for gi, group, arena, todo in work:
            with _lib.on_device(arena.index):
                self._step_group(gi, group, arena, todo)
        return loss

    def _salt(self, gi):
        return (self.seed * _SALT_SEED + gi * _SALT_GROUP) & 0xFFFFFFFF

    @staticmethod
    def _touched(tensors):
        """Marked as modified in place: a step writes through addresses."""
        if _lib.torch_fn("pin_torch_touched")(tensors) != 0:
            raise RuntimeError("AdamW: a parameter is not a tensor")

    def _step_group(self, gi, group, arena, todo):
        lr, (b1, b2) = group["lr"], group["betas"]
        stream = _lib.stream(arena.index)
        wd, salt = float(group["weight_decay"]), self._salt(gi)
        lr_dev = lr if isinstance(lr, torch.Tensor) and self.capturable else None
        rates = (0.0 if lr_dev is not None else float(lr), float(b1), float(b2))
        if self.capturable:
            _lib.call("pin_adamw_scalars", _lib.ptr(arena.step_dev), _lib.ptr(lr_dev), *rates, wd, salt,
                      _lib.ptr(arena.scalars), stream)
        for idx, dtype, ps, gs in todo:
            if idx is None:
                written = group["params"]
                n, sizes, offsets = len(ps), arena.c_sizes, arena.c_offsets
            else:
                written = [group["params"][i] for i in idx]
                n = len(idx)
                sizes, offsets = (array("q", [x[i] for i in idx]) for x in (arena.sizes, arena.offsets))
            t = arena.steps[0 if idx is None else idx[0]] + (0 if self.capturable else 1)
            master = arena.master if dtype != torch.float32 else None
            try:
                _lib.call("pin_adamw_step", ps.buffer_info()[0], gs.buffer_info()[0], sizes.buffer_info()[0],
                          offsets.buffer_info()[0], n, _lib.TYPES[dtype], arena.bits, _lib.ptr(arena.m), _lib.ptr(arena.v),
                          _lib.ptr(arena.exps), _lib.ptr(master), arena.total, *rates, float(group["eps"]), wd, t, salt,
                          _lib.ptr(arena.scalars), stream)
            finally:   # (while the kernels run)
                self._touched(written + arena.written)
            if self.capturable:
                continue
            if idx is None:
                arena.steps = [t] * n
            else:
                for i in idx:
                    arena.steps[i] = t
                arena.together = len(set(arena.steps)) == 1
        arena.held = None

    def _seen(self, gi):
        """What there is of a group's state; before its first step what that would find, which is not kept (a copy of the
        parameters that is made here would miss what they are changed to before it)."""
        group = self.param_groups[gi]
        if gi % len(self.param_groups) in self._arenas and group["params"][0] in self.state:
            return self._arena(gi)
        for p in group["params"]:
            _lib.require_device(p)
        return _Arena(group, False)

    def offsets(self, group=0):
        """First element of each parameter of the group in the flat arrays."""
        return list(self._seen(group).offsets)

    def moments(self, group=0):
        """Both moments of a parameter group as flat float32 arrays (of 8-bit state: the values that
        its codes stand for; of 32-bit state: the state itself)."""
        arena = self._seen(group)
        if arena.bits == 32:
            return arena.m, arena.v
        m = torch.empty((arena.total,), dtype=torch.float32, device=arena.device)
        v = torch.empty_like(m)
        with _lib.on_device(arena.index):
            _lib.call("pin_adamw_moments", _lib.ptr(arena.m), _lib.ptr(arena.v), _lib.ptr(arena.exps), arena.total,
                      _lib.ptr(m), _lib.ptr(v), _lib.stream(arena.index))
        return m, v

    def master(self, group=0):
        """The group's parameters in 32 bits as one flat array (None without master_weights)."""
        return self._seen(group).master

    def state_dict(self):
        kept = dict(self.state)
        for gi, arena in self._arenas.items():
            step = None if arena.step_dev is None else int(arena.step_dev)
            for p, n in zip(self.param_groups[gi]["params"], arena.steps):   # the counts as torch's hooks expect them
                if p in kept:
                    self.state[p] = {"step": n if step is None else step, **kept[p]}
        try:
            return super().state_dict()
        finally:
            self.state.update(kept)

    def load_state_dict(self, state_dict):
        """Takes a state_dict of an AdamW with the same groups (its state_bits and master_weights too).  State that is
        there already is written where it lies, so a graph that holds a step goes on from what was loaded.  torch's
        hooks of loading and saving run as they do around its own optimisers."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        if "state" not in state_dict or "param_groups" not in state_dict:
            raise ValueError("AdamW: the saved state has no state or no param_groups: not an optimiser's")
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the saved state has other parameter groups")
        for mine, saved in zip(self.param_groups, groups):
            for key in _RATES:
                if key not in saved:
                    raise ValueError(f"AdamW: the saved state's groups have no {key} (another optimiser's?)")
            for key in ("state_bits", "master_weights"):
                if mine[key] != saved[key]:
                    raise ValueError(f"AdamW: the saved state has {key} {saved[key]}, this optimiser {mine[key]}")
            self._check_rates(saved, float(saved["lr"]))
        plan = []
        k = 0
        for gi, group in enumerate(self.param_groups):
            for i, p in enumerate(group["params"]):
                one = state_dict["state"].get(groups[gi]["params"][i])
                k += 1
                if one is None:
                    continue
                want = [*_STATE_KEYS[group["state_bits"]]] + ["master"] * _has_master(group)
                kind = torch.float32 if group["state_bits"] == 32 else torch.uint8
                for key in want:
                    shape = (_blocks(p.numel()), 2) if key == "exponents" else tuple(p.shape)
                    dtype = {"exponents": torch.int16, "master": torch.float32}.get(key, kind)
                    if key not in one or tuple(one[key].shape) != shape or one[key].dtype != dtype:
                        raise ValueError(f"AdamW: the saved {key} of parameter {k - 1} is not a {dtype} of {shape}")
                if int(one.get("step", -1)) < 0:
                    raise ValueError(f"AdamW: the saved step of parameter {k - 1} is {one.get('step')}")
                plan.append((gi, i, p, want, one))
            if self.capturable and len({int(o["step"]) for g, _, _, _, o in plan if g == gi}) > 1:
                raise ValueError("AdamW: with capturable=True the parameters of a group share one step")
        # the optimiser's own state_dict is views of what is started anew here
        own = {x.untyped_storage().data_ptr() for arena in self._arenas.values() for x in arena.arrays()}
        plan = [(gi, i, p, want, {key: x.clone() if key in want and x.untyped_storage().data_ptr() in own else x
                                  for key, x in one.items()}) for gi, i, p, want, one in plan]
        for gi, group in enumerate(self.param_groups):
            arena = self._arenas.get(gi)
            if arena is None:
                continue
            if arena.fits(group):
                arena.start(group["params"])
            else:
                del self._arenas[gi]
                for p in group["params"]:
                    self.state.pop(p, None)
        for mine, saved in zip(self.param_groups, groups):
            lr = float(saved["lr"])
            if isinstance(mine["lr"], torch.Tensor):   # (a graph may read it)
                lr = mine["lr"].fill_(lr)
            mine.update({key: val for key, val in saved.items() if key != "params"}, lr=lr)
        to, by = {}, {}
        for gi, i, p, want, one in plan:
            arena = self._arena(gi)
            for key in want:
                pair = to.setdefault((gi, one[key].dtype, one[key].device), ([], []))
                pair[0].append(self.state[p][key])
                pair[1].append(one[key])
            arena.steps[i] = int(one["step"])
            if arena.step_dev is not None:
                by[gi] = arena.steps[i]
        for mine, saved in to.values():
            torch._foreach_copy_(mine, saved)
        for arena in self._arenas.values():
            arena.together = len(set(arena.steps)) == 1
        for gi, step in by.items():
            self._arenas[gi].step_dev.fill_(step)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)
