"""AdamW over many tensors where they lie: `MultiTensorAdamW`, a torch optimizer on the HIP kernels of csrc/multi_adamw.hip.

`train.FlatAdamW` updates ONE flat fp32 buffer that every parameter was re-homed into.  This one takes the parameters as they
are -- fp32, bf16 or fp16, frozen ones among them, convolution weights in channels_last, optionally with fp32 masters behind
16-bit weights -- and holds their moments in 32 or in 8 bits.  Step counts live on the device, so a captured step goes on
counting when it is replayed."""
import ctypes

import torch
from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from . import _lib
from .ops import _ptr

BLOCK = 32                      # elements that share an exponent byte (8-bit moments); tensors start at multiples of it
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ZERO_EXPONENT = 16             # exponent byte of a block of zeros


def _dense(t):
    """Non-overlapping and dense in some order of its dimensions (contiguous, channels_last, a transpose of either)."""
    if t.numel() == 0 or t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _memory_order(t):
    """The dimensions of a dense tensor from the slowest in memory to the fastest, without those of one element."""
    if t.numel() == 0:
        return []
    return [d for _, d in sorted(((-t.stride(d), d) for d in range(t.dim()) if t.shape[d] != 1))]


class MultiTensorAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay) of all parameters in two launches per 384 tensors, whatever their sizes.

    params: tensors or parameter groups (lr, betas, eps, weight_decay per group); all on one GPU, each dense (in any order of
    its dimensions), float32 / bfloat16 / float16.  A group's lr may be a 0-d float32 tensor on that GPU: a captured step then
    reads it at every replay.
    state_bits: 32 = moments in fp32; 8 = one byte per moment and element plus one exponent byte for 32 elements, rounded
    stochastically (reproducibly: a function of seed, parameter index, step and element).  The second moment is held as its root.
    master_weights: keep an fp32 copy of every 16-bit parameter and update that; the parameter is its rounding.  Without
    it a 16-bit parameter is updated in place and rounded to nearest, as torch.optim.AdamW does.  Whoever else writes such a
    parameter (a checkpoint loaded into the model alone) calls sync_masters().

    The defaults are the pre-training config's (lr 1e-5, weight_decay 0.05).  Gradients are read where they are when step() is
    called; parameters without one are skipped and do not count the step."""

    def __init__(self, params, lr=1e-5, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05, state_bits=32, master_weights=False,
                 seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        self._check_hyper(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.master_weights, self.seed = int(state_bits), bool(master_weights), int(seed)
        if not 0 <= self.seed < 2 ** 32:
            raise ValueError("seed must be in [0, 2**32)")
        self._arena, self._building, self._plan, self._layout, self._retired = None, True, None, [], []
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        if not self._params():
            raise ValueError("MultiTensorAdamW: no parameter in any group")
        self._building = False
        self._build()

    # ------------------------------------------------------------------------------------------------ construction
    @staticmethod
    def _check_hyper(g):
        b1, b2 = g["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {g['betas']}")
        if g["eps"] < 0.0 or g["weight_decay"] < 0.0 or (not torch.is_tensor(g["lr"]) and g["lr"] < 0.0):
            raise ValueError(f"lr, eps and weight_decay must not be negative, got {g['lr']}, {g['eps']}, {g['weight_decay']}")

    def add_param_group(self, group):
        """A refused group leaves the optimizer as it was.  A step that was captured before goes on with the state of that time:
        capture it anew."""
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_hyper(g)
            if torch.is_tensor(g["lr"]) and (g["lr"].dtype != torch.float32 or g["lr"].numel() != 1 or not g["lr"].is_cuda):
                raise ValueError("a tensor lr must be one float32 value on the GPU")
            self._check_params(g["params"])
            self._check_apart()
            if not self._building:
                self._build()
        except Exception:
            self.param_groups.pop()
            raise

    def _check_params(self, params):
        if not self._params():
            return                                  # (a group without parameters, e.g. of a model without biases; the next ones have some)
        first = self._params()[0]
        if len({id(p) for p in params}) != len(params):
            raise ValueError("MultiTensorAdamW: a parameter is listed twice")
        for p in params:
            if not p.is_cuda:
                raise RuntimeError("MultiTensorAdamW: parameters must be CUDA tensors (geomae_amd has no CPU path)")
            if p.device != first.device:
                raise RuntimeError(f"MultiTensorAdamW: parameters on {first.device} and on {p.device}: one optimizer per GPU")
            if p.dtype not in _DTYPE:
                raise RuntimeError(f"MultiTensorAdamW: parameters must be float32, bfloat16 or float16, got {p.dtype}")
            if p.layout != torch.strided or not _dense(p):
                raise RuntimeError("MultiTensorAdamW: parameters must be dense (no gaps or overlaps between their elements)")

    def _check_apart(self):
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self._params() if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("MultiTensorAdamW: two parameters share memory")

    def _params(self):
        return [p for g in self.param_groups for p in g["params"]]

    def _build(self):
        """Moments of all parameters in one arena per kind, each parameter's part starting at a multiple of 32 elements; a
        parameter's state tensors are views of it in the parameter's own layout.  Parameters that were there keep theirs.  Nothing
        of the optimizer changes before all of it is there."""
        params, had = self._params(), len(self._layout)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("MultiTensorAdamW: parameters cannot be added while a stream is captured")
        if had:
            self._check_layout([p for g in self.param_groups[:-1] for p in g["params"]])
        dev = params[0].device
        torch.cuda.synchronize(dev)                 # (steps of any stream, whose state is copied below)
        offsets, total = [], 0
        for p in params:
            offsets.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        kind = torch.float32 if self.state_bits == 32 else torch.uint8
        arena = {"exp_avg": torch.zeros(total, dtype=kind, device=dev), "exp_avg_sq": torch.zeros(total, dtype=kind, device=dev),
                 "step": torch.zeros(len(params), dtype=torch.int64, device=dev)}
        if self.state_bits == 8:
            for k in ("exp_avg_exponent", "exp_avg_sq_exponent"):
                arena[k] = torch.full((total // BLOCK,), _ZERO_EXPONENT, dtype=torch.uint8, device=dev)
        if self.master_weights:
            arena["master"] = torch.zeros(total, dtype=torch.float32, device=dev)
        state = [self._views(arena, i, p, off) for i, (p, off) in enumerate(zip(params, offsets))]
        for i, (p, new) in enumerate(zip(params, state)):
            for k, v in new.items():
                if i < had:
                    v.copy_(self.state[p][k])
                elif k == "master":
                    v.copy_(p.detach())
        lib = _lib.load()
        chunk = lib.geomae_multi_adamw_chunk()
        counts = [-(-p.numel() // chunk) for p in params]
        first = [0]
        for c in counts:
            first.append(first[-1] + c)
        tensor = torch.repeat_interleave(torch.arange(len(params), dtype=torch.int32), torch.tensor(counts, dtype=torch.int64))
        within = torch.arange(first[-1], dtype=torch.int64) - torch.tensor(first[:-1], dtype=torch.int64)[tensor.long()]
        chunks = torch.stack([tensor, within.int()], 1).contiguous().to(dev)
        workspace = torch.empty(lib.geomae_multi_adamw_workspace_bytes(len(params)), dtype=torch.uint8, device=dev)
        norm_word = torch.zeros((), dtype=torch.float32, device=dev)
        torch.cuda.synchronize(dev)                 # (the first step may be on any stream)
        self._set_table(params, arena, offsets, chunks, first, workspace, norm_word)
        self.state.update(zip(params, state))

    def _retire(self):
        """What a captured step may still read and write is kept as long as this optimizer."""
        if self._plan is not None and self._plan.captured:
            self._retired.append((self._table, self._arena, self._chunks, self._workspace, self._norm_word))

    @staticmethod
    def _part(flat, off, p):
        """p's own part of an arena, in p's layout."""
        return flat.as_strided(p.shape, p.stride(), off) if p.numel() else flat[off:off].view(p.shape)

    def _views(self, arena, i, p, off):
        blocks = slice(off // BLOCK, off // BLOCK + -(-p.numel() // BLOCK))
        out = {"step": arena["step"][i]}
        for k in ("exp_avg", "exp_avg_sq"):
            out[k] = self._part(arena[k], off, p)
            if self.state_bits == 8:
                out[k + "_exponent"] = arena[k + "_exponent"][blocks]
        if self.master_weights and p.dtype != torch.float32:
            out["master"] = self._part(arena["master"], off, p)
        return out

    def _set_table(self, params, arena, offsets, chunks, first_chunk, workspace, norm_word):
        """Take these buffers, with a device table of the addresses in them."""
        rows = (_lib.GeomaeAdamwTensor * len(params))()
        item = arena["exp_avg"].element_size()
        for i, (p, off) in enumerate(zip(params, offsets)):
            r = rows[i]
            r.param = p.data_ptr()
            r.exp_avg, r.exp_avg_sq = arena["exp_avg"].data_ptr() + off * item, arena["exp_avg_sq"].data_ptr() + off * item
            if self.state_bits == 8:
                r.exp_avg_exponent = arena["exp_avg_exponent"].data_ptr() + off // BLOCK
                r.exp_avg_sq_exponent = arena["exp_avg_sq_exponent"].data_ptr() + off // BLOCK
            r.master = arena["master"].data_ptr() + 4 * off if self.master_weights and p.dtype != torch.float32 else None
            r.step = arena["step"].data_ptr() + 8 * i
            r.numel, r.dtype, r.index = p.numel(), _DTYPE[p.dtype], i
        table = torch.frombuffer(bytearray(rows), dtype=torch.uint8).to(params[0].device)
        plan = _lib.host().AdamwPlan(params, first_chunk, table.data_ptr(), chunks.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                     norm_word.data_ptr(), self.state_bits)
        self._retire()
        self._arena, self.offsets, self._chunks, self._first_chunk = arena, offsets, chunks, first_chunk
        self._workspace, self._norm_word, self._table, self._plan = workspace, norm_word, table, plan
        self._layout = self._layouts(params)

    @staticmethod
    def _layouts(params):
        return [(id(p), p.shape, p.stride(), p.dtype, p.device) for p in params]

    def _check_layout(self, params):
        if [l[0] for l in self._layouts(params)] != [l[0] for l in self._layout]:
            raise RuntimeError("MultiTensorAdamW: a parameter was replaced, removed or moved in its groups (the moments would be another's); "
                               "make a new optimizer")
        if self._layouts(params) != self._layout:
            raise RuntimeError("MultiTensorAdamW: a parameter changed its shape, layout, dtype or device; make a new optimizer")

    # ------------------------------------------------------------------------------------------------ the step
    def step(self, closure=None, max_norm=0.0, grad_scale=1.0, skip_nonfinite=False):
        """One update of every parameter that has a gradient.  max_norm > 0 clips the gradients to that norm over all of
        them (torch.nn.utils.clip_grad_norm_; infinity: only the norm is wanted; 0 or None: no clipping); grad_scale (a number, or one
        float32 value on the GPU) multiplies them first;
        skip_nonfinite leaves everything as it was if their norm is not finite.  After a step with max_norm or
        skip_nonfinite, `grad_norm` is the scaled gradients' norm before clipping (a 0-d tensor that the next step
        overwrites).  Gradients are not changed."""
        # (a class that overrides step() is wrapped itself)
        if type(self).step is MultiTensorAdamW.step and (
                self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_optimizer_pre_hooks
                or _global_optimizer_post_hooks or torch.autograd._profiler_enabled()):
            return self._observed_step(closure, max_norm, grad_scale, skip_nonfinite)
        return self._step(closure, max_norm, grad_scale, skip_nonfinite)

    # torch wraps step() of every optimizer for hooks and the profiler, 5 us on the host where a step of few tensors takes 9: here
    # the wrapper is gone through when there is a hook or a profiler
    step.hooked = True

    def _step(self, closure=None, max_norm=0.0, grad_scale=1.0, skip_nonfinite=False):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        scale, scale_tensor = (1.0, grad_scale) if torch.is_tensor(grad_scale) else (float(grad_scale), None)
        max_norm = float(max_norm or 0.0)
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        if len(self.state) < len(self._layout):
            raise RuntimeError("MultiTensorAdamW: the state was cleared or replaced, which does not reach the moments; load a state_dict (one with an "
                               "empty state begins anew)")
        self._plan.seed = self.seed
        if not self._plan.step(self.param_groups, max_norm, scale, scale_tensor, skip_nonfinite):
            self._find_params()
            if not self._plan.step(self.param_groups, max_norm, scale, scale_tensor, skip_nonfinite):
                raise RuntimeError("MultiTensorAdamW: the parameters moved during the step")
        if self._plan.new_stream:                   # the caller knows nothing of these: their memory waits for this stream by itself
            for t in (self._table, self._chunks, self._workspace, self._norm_word, *self._arena.values()):
                t.record_stream(torch.cuda.current_stream(t.device))
        if max_norm > 0.0 or skip_nonfinite:
            self.grad_norm = self._norm_word
        return loss

    _observed_step = torch.optim.Optimizer.profile_hook_step(_step)

    def _find_params(self):
        """A parameter is not where or what the device table says: make the table anew."""
        params = self._params()
        self._check_layout(params)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("MultiTensorAdamW: a parameter's storage moved; take one step outside the capture first")
        self._check_params(params)
        self._check_apart()
        self._set_table(params, self._arena, self.offsets, self._chunks, self._first_chunk, self._workspace, self._norm_word)

    # ------------------------------------------------------------------------------------------------ state
    def moments(self):
        """(first, second moment) of all parameters as two flat tensors, parameter i's from self.offsets[i] on in its memory
        order.  32 bits: the fp32 moments themselves (not a copy).  8 bits: the values that the codes stand for, in bfloat16
        (which holds them exactly), the second as the root that is stored."""
        a = self._arena
        if self.state_bits == 32:
            return a["exp_avg"], a["exp_avg_sq"]
        n, dev = a["exp_avg"].numel(), a["exp_avg"].device
        out = [torch.empty(n, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        with torch.cuda.device(dev):
            _lib.check(_lib.load().geomae_adamw_moments8(
                _ptr(a["exp_avg"]), _ptr(a["exp_avg_exponent"]), _ptr(a["exp_avg_sq"]), _ptr(a["exp_avg_sq_exponent"]), n,
                _ptr(out[0]), _ptr(out[1]), ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "geomae_adamw_moments8")
        return out[0], out[1]

    def masters(self):
        """The fp32 masters as one flat tensor (not a copy), parameter i's from self.offsets[i] on; fp32 parameters have none."""
        if not self.master_weights:
            raise RuntimeError("MultiTensorAdamW: made without master_weights")
        return self._arena["master"]

    def steps(self):
        """The steps that each parameter has taken, as an int64 tensor (not a copy)."""
        return self._arena["step"]

    @torch.no_grad()
    def sync_masters(self):
        """Take the masters from the parameters."""
        for p in self._params():
            if "master" in self.state[p]:
                self.state[p]["master"].copy_(p)

    def load_flat_state(self, state, step):
        """Fill the moments (and masters) from flat tensors laid out as moments() and masters() give them -- at 8 bits the codes
        and their exponent bytes -- and set every parameter's step count."""
        if set(state) != set(self._arena) - {"step"}:
            raise ValueError(f"flat state must have {sorted(set(self._arena) - {'step'})}, got {sorted(state)}")
        for k, v in state.items():
            if v.shape != self._arena[k].shape or v.dtype != self._arena[k].dtype:
                raise ValueError(f"flat state {k}: {tuple(v.shape)} {v.dtype}, expected {tuple(self._arena[k].shape)} {self._arena[k].dtype}")
        for k, v in state.items():
            self._arena[k].copy_(v)
        self._arena["step"].fill_(int(step))

    def __getstate__(self):
        raise TypeError("a MultiTensorAdamW holds device addresses and cannot be copied or pickled: keep its state_dict()")

    def state_dict(self):
        sd = super().state_dict()
        sd["state_bits"], sd["master_weights"], sd["seed"] = self.state_bits, self.master_weights, self.seed
        if self.state_bits == 8:
            # an exponent byte belongs to 32 codes in memory order, whatever order a saved tensor of codes has by the time it is loaded
            sd["memory_orders"] = [_memory_order(p) for p in self._params()]
        return sd

    def load_state_dict(self, sd):
        """A state_dict of this class with the same state_bits and masters, or (32 bits) one of torch.optim.AdamW.  Parameters
        that it has no state of begin anew; masters that it does not hold are taken from the parameters.  An 8-bit state of a parameter
        in another memory order (contiguous, now channels_last) is refused: its blocks are other elements here."""
        sd = dict(sd)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            new = hook(self, sd)
            sd = sd if new is None else new
        self.check_state(sd)()
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def check_state(self, sd):
        """ValueError if load_state_dict() would refuse this state; else the function that takes it."""
        if int(sd.get("state_bits", 32)) != self.state_bits:
            raise ValueError(f"the state holds moments in {sd.get('state_bits', 32)} bits, this optimizer in {self.state_bits}")
        groups = sd["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state's parameter groups do not match this optimizer's")
        if any(g.get("amsgrad") or g.get("maximize") for g in groups):
            raise ValueError("amsgrad and maximize are not supported")
        params, ids = self._params(), [i for g in groups for i in g["params"]]
        todo, orders = [], sd.get("memory_orders")
        if orders is not None and len(orders) != len(params):
            raise ValueError(f"the state has memory orders of {len(orders)} parameters, this optimizer has {len(params)}")
        for n, (p, i) in enumerate(zip(params, ids)):
            st, mine = sd["state"].get(i), self.state[p]
            if st is not None and self.state_bits == 8 and "exp_avg" in st and "exp_avg_sq" in st:
                for k in ("exp_avg", "exp_avg_sq"):
                    order = _memory_order(st[k]) if orders is None else list(orders[n])
                    if order != _memory_order(p):
                        raise ValueError(f"the state of parameter {i}: {k} has codes with the dimensions in memory order {order}, the "
                                         f"parameter {_memory_order(p)}; their exponents are of 32 neighbours in memory")
            if st is None:
                st = {k: torch.full((), _ZERO_EXPONENT if k.endswith("exponent") else 0, dtype=v.dtype).expand(v.shape)
                      for k, v in mine.items() if k != "master"}
            for k, v in mine.items():
                if k == "master" and k not in st:
                    todo.append((v, p.detach()))
                    continue
                if k not in st:
                    raise ValueError(f"the state of parameter {i} has no {k}")
                x = st[k] if torch.is_tensor(st[k]) else torch.tensor(st[k])
                if k != "step" and (x.shape != v.shape or (x.dtype == torch.uint8) != (v.dtype == torch.uint8)):
                    raise ValueError(f"the state of parameter {i}: {k} is {tuple(x.shape)} {x.dtype}, expected {tuple(v.shape)} {v.dtype}")
                todo.append((v, x.reshape(v.shape)))
        for g, h in zip(self.param_groups, groups):
            self._check_hyper({**g, **{k: v for k, v in h.items() if k != "params"}})

        @torch.no_grad()
        def take():
            for v, x in todo:
                v.copy_(x)
            for g, h in zip(self.param_groups, groups):
                mine, lr = g["lr"], float(h.get("lr", g["lr"]))
                g.update({k: v for k, v in h.items() if k != "params"})
                g["lr"] = mine.fill_(lr) if torch.is_tensor(mine) else lr   # (a captured step reads a tensor lr where it is)
            self.seed = int(sd.get("seed", self.seed))
        return take
