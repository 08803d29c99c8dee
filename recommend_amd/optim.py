"""The optimizers on the library's kernels: FusedClipAdam, and FusedAdamW (rk_adamw_step; described there).

FusedClipAdam is Adam with global-norm gradient clipping on the two-launch kernel pair
(rk_adam_clip_step_f32): the optimizer half of train/graph_trainer.py:151-156,
`clip_grad_norm_(model.parameters(), max_norm); optimizer.step()`, for fp32 parameters.

The update is torch.optim.Adam's (same constants, same order of operations); moments and the step
count live in device memory, the learning rate is a device scalar refreshed from
`param_groups[0]['lr']`, so a step captured in a HIP graph keeps working when a scheduler changes
the rate between replays.  Parameters whose `.grad` is None take no part, as in torch.

Checkpoints (train/graph_trainer.py:279,315 save and restore `optimizer.state_dict()`): the state
dict carries `step`, `exp_avg`, `exp_avg_sq` per parameter exactly as torch.optim.Adam's does, so a
checkpoint written by either optimizer loads into the other and a resumed run continues the bias
correction where it stopped.

Several GPUs: parameters listed in `sharded_params` are row shards (every rank holds other rows);
their squared gradient norms are summed over the ranks of `group` by one all-reduce of one float
between the two launches (rk_adam_sqnorm_f32 / rk_adam_update_f32).  All other parameters are
taken to be replicated with gradients already summed over the ranks."""
import torch

from . import _ffi
from ._ffi import c_float, c_int32, ptr, stream_ptr

_MAX_TABLES = 4     # descriptor tables kept (one per set of gradient buffers: eager steps, a captured graph)


class FusedClipAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, max_grad_norm=None,
                 sharded_params=None, group=None, all_reduce=None):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        if len(self.param_groups) != 1:
            raise ValueError("FusedClipAdam takes one parameter group")
        self.max_grad_norm = max_grad_norm
        self._sharded = {id(p) for p in (sharded_params or [])}
        self._group = group
        self._all_reduce = all_reduce    # all_reduce(tensor, group): sums in place (default: torch.distributed)
        self._tables = {}        # pointer set -> (descriptor array, workspace, replicated count)
        self._held = []          # memory that a step recorded in a HIP graph may go on using
        self._dev = None
        self._lr_host = None
        self._restored_step = None
        self.grad_norm = None    # device scalar: total gradient norm of the last step, before clipping

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables = {}
        self.__dict__.setdefault("_held", [])

    def _state_for(self, p):
        st = self.state[p]
        if "exp_avg" not in st:
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        return st

    def _init_device(self, dev):
        self._dev = dev
        self.step_count = torch.full((1,), int(self._restored_step or 0), dtype=torch.int64, device=dev)
        self.lr_dev = torch.zeros(1, dtype=torch.float32, device=dev)
        self.grad_norm = torch.zeros(1, dtype=torch.float32, device=dev)
        self.shard_sq = torch.zeros(1, dtype=torch.float32, device=dev)

    def _prepare(self, params):
        """Descriptor table + workspace for this set of parameter / gradient / moment buffers
        (replicated tensors first, row shards behind them)."""
        states = [self._state_for(p) for p in params]
        key = tuple((p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), p.numel())
                    for p, st in zip(params, states))
        tab = self._tables.get(key)
        if tab is None:
            order = sorted(range(len(params)), key=lambda i: id(params[i]) in self._sharded)   # stable
            arr = (_ffi.AdamTensor * len(params))()
            for j, i in enumerate(order):
                p, st = params[i], states[i]
                arr[j] = _ffi.AdamTensor(p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(),
                                         st["exp_avg_sq"].data_ptr(), p.numel())
            n_rep = sum(1 for p in params if id(p) not in self._sharded)
            nbytes = _ffi.load().rk_adam_ws_bytes(arr, len(params))
            tab = (arr, torch.empty(nbytes // 4 + 4, dtype=torch.float32, device=self._dev), n_rep)
            while len(self._tables) >= _MAX_TABLES:         # oldest first: dicts keep insertion order
                self._tables.pop(next(iter(self._tables)))
            self._tables[key] = tab
        return tab

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        group = self.param_groups[0]
        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return loss
        for p in params:
            if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() and p.grad.is_contiguous()
                    and p.grad.dtype == torch.float32):
                raise _ffi.RkError(_ffi.RK_ERR_UNSUPPORTED, "FusedClipAdam: contiguous fp32 parameters and gradients "
                                   "on a HIP device only")
        if self._dev is None:
            self._init_device(params[0].device)
        arr, ws, n_rep = self._prepare(params)     # (moments are created outside any graph capture: first eager step)
        if torch.cuda.is_current_stream_capturing():
            self._held.append(ws)                  # (the table that holds it may go before the graph does)
        if self._lr_host != group["lr"]:
            if torch.cuda.is_current_stream_capturing():
                if self._lr_host is None:
                    raise RuntimeError("run one optimizer step before capturing it in a graph")
            else:
                self.lr_dev.fill_(float(group["lr"]))
                self._lr_host = group["lr"]
        b1, b2 = group["betas"]
        n = len(params)
        max_norm = c_float(self.max_grad_norm if self.max_grad_norm else 0.0)
        if n_rep == n:
            _ffi.call("rk_adam_clip_step_f32", arr, c_int32(n), ptr(self.step_count), ptr(self.lr_dev),
                      c_float(b1), c_float(b2), c_float(group["eps"]), c_float(group["weight_decay"]),
                      max_norm, ptr(self.grad_norm), ptr(ws), _ffi.c_size_t(ws.numel() * 4), stream_ptr(self._dev))
            return loss
        _ffi.call("rk_adam_sqnorm_f32", arr, c_int32(n), c_int32(n_rep), ptr(self.step_count), ptr(self.shard_sq),
                  ptr(ws), _ffi.c_size_t(ws.numel() * 4), stream_ptr(self._dev))
        if self._all_reduce is not None:
            self._all_reduce(self.shard_sq, self._group)
        else:
            import torch.distributed as dist
            if dist.is_initialized() and dist.get_world_size(self._group) > 1:
                dist.all_reduce(self.shard_sq, group=self._group)
        _ffi.call("rk_adam_update_f32", arr, c_int32(n), c_int32(n_rep), ptr(self.step_count), ptr(self.lr_dev),
                  c_float(b1), c_float(b2), c_float(group["eps"]), c_float(group["weight_decay"]), max_norm,
                  ptr(self.shard_sq), ptr(self.grad_norm), ptr(ws), _ffi.c_size_t(ws.numel() * 4),
                  stream_ptr(self._dev))
        return loss

    def state_dict(self):
        """torch.optim.Adam's layout: every parameter's state carries `step` beside its moments
        (reading the device counter synchronises)."""
        if self._dev is not None:
            t = float(self.step_count.item())
            for st in self.state.values():
                if "exp_avg" in st:
                    st["step"] = torch.tensor(t)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """Moments and step count of a checkpoint (this optimizer's or torch.optim.Adam's).  Moment
        buffers that exist already keep their memory and take the checkpoint's VALUES (zeros, where it has
        none for their parameter), so a training step recorded in a HIP graph before the load (its kernels
        hold the buffers' addresses) goes on updating the moments the optimizer reports; the learning rate of
        the checkpoint reaches the device scalar at once for the same reason.  Call it outside graph capture."""
        old = {p: (st["exp_avg"], st["exp_avg_sq"]) for p, st in self.state.items() if "exp_avg" in st}
        super().load_state_dict(state_dict)
        for q, (m, v) in old.items():
            st = self.state.get(q)
            if st is None or "exp_avg" not in st:
                m.zero_()
                v.zero_()
                self.state[q] = {"exp_avg": m, "exp_avg_sq": v}
            elif st["exp_avg"].shape == m.shape and st["exp_avg"].device == m.device:
                m.copy_(st["exp_avg"])
                v.copy_(st["exp_avg_sq"])
                st["exp_avg"], st["exp_avg_sq"] = m, v
            else:
                self._held += [m, v]
        self._tables = {}        # descriptor tables are rebuilt from the state at the next step
        steps = [float(st["step"]) for st in self.state.values() if "step" in st]
        self._restored_step = int(max(steps)) if steps else 0
        if self._dev is not None:
            self.step_count.fill_(self._restored_step)
        self._lr_host = None
        self.sync_lr()

    def sync_lr(self):
        """Push a learning rate changed by a scheduler to the device scalar.  step() does it, and so do the recorded steps
        of train_step and dist_train; call it before replaying a graph of your own, outside the capture."""
        lr = self.param_groups[0]["lr"]
        if self._dev is not None and self._lr_host != lr:
            self.lr_dev.fill_(float(lr))
            self._lr_host = lr


_FULL = 448.0       # largest finite e4m3 value
_TINY = 1e-30       # block maxima below this count as this
_STATE32 = ("exp_avg", "exp_avg_sq")
_STATE8 = ("exp_avg8", "exp_avg8_scale", "exp_avg_sq8", "exp_avg_sq8_scale")


def encode_moment(x, keep_above_zero=False):
    """fp32 values -> (e4m3 codes padded to whole blocks of 64, one fp32 scale per block), the form in which
    FusedAdamW holds 8-bit moments: value = code * scale.  keep_above_zero: positive values get at least
    the smallest code (the root of a second moment)."""
    x = x.detach().float().reshape(-1)
    x = torch.nn.functional.pad(x, (0, -x.numel() % _ffi.ADAMW_BLOCK)).view(-1, _ffi.ADAMW_BLOCK)
    most = x.abs().amax(1, keepdim=True).clamp_min(_TINY)
    y = x * (most.reciprocal() * _FULL)
    if keep_above_zero:
        y = torch.where(x > 0, y.clamp_min(2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).view(-1), (most * (1.0 / _FULL)).view(-1)


def decode_moment(code, scale, like):
    """The fp32 values that codes and scales stand for, in the shape of the parameter `like`."""
    return (code.float().view(-1, _ffi.ADAMW_BLOCK) * scale.unsqueeze(1)).view(-1)[:like.numel()].view(like.shape)


_NEVER = 2 ** 62        # elements that no tensor has


def _not_in_a_capture():
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("run one optimizer step with these parameters before capturing it in a graph")


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (the reference trainer's other choice, train/graph_trainer.py:78-101) with
    clip_grad_norm_ on the library's fused step (rk_adamw_step), over all parameter groups at once.

    Parameters and gradients: contiguous fp32, bfloat16 or fp16 on one HIP device (gradients in the
    parameter's type or fp32); the arithmetic is fp32 and a parameter is rounded once.  Up to
    8 parameter groups with their own lr, betas, eps and weight_decay.

    state_bits=32: fp32 moments, torch.optim.AdamW's state (`step`, `exp_avg`, `exp_avg_sq`).
    state_bits=8: tensors of at least `min_8bit_size` elements hold exp_avg and the root of exp_avg_sq as
    torch.float8_e4m3fn codes with one fp32 scale per 64 consecutive elements (`exp_avg8`,
    `exp_avg8_scale`, `exp_avg_sq8`, `exp_avg_sq8_scale`): 2.1 bytes for each element instead of 8.

    What 8-bit moments do not follow: codes are rounded to nearest after every step, so a root changes its code only
    where one step moves it by half a code (3 to 6 %) against the largest of its block of 64.  With betas[1] = 0.999 a
    step takes at most 0.05 % off a root: against its block it never falls, and rises only for gradients several
    times as large.  Simulated, 4,000 steps, scales of a block's elements spread by e^1, against 32-bit moments:
      steady gradients                          cosine of the update 0.988, roots (99.8 % of them) 0.67 to 1.70 times
      all gradients a tenth from step 500 on    the same: a block's scale follows
      every second element's a tenth            cosine 0.96, 0.88, 0.80 at step 1,000, 2,000, 4,000, the update's norm up to
                                                1.96 times; their roots 5.7 times too large (median; their rate is too
                                                small by that), their neighbours' down to 0.24 of what they should be
      every second element's threefold          cosine 0.85; the others' roots 2.4 times too large, theirs down to 0.35
    The third case with betas[1] = 0.99: 0.82, with 0.95: 0.996.  Where the scales of neighbouring elements come apart
    during training take state_bits=32 (or a min_8bit_size that leaves those tensors out), or betas[1] up to 0.95.

    As with FusedClipAdam the step count and the learning rates live in device memory, a step can be
    recorded in a HIP graph after one eager step, and parameters without a gradient take no part.  The
    step count is one for all parameters, where torch.optim.AdamW counts each one's own: a parameter whose first
    gradient comes late is corrected with the count of the others (with the default betas its first updates are up to
    (1 - beta1) / (1 - beta2)^(1/2) = 3.2 times as large), and a checkpoint whose counts differ continues with the
    largest.  Parameters must not share memory (one object given twice in a group
    is refused).  Checkpoints load across state_bits and from torch.optim.AdamW."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=None,
                 state_bits=32, min_8bit_size=4096):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, not {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.max_grad_norm = max_grad_norm
        self.state_bits = state_bits
        self.min_8bit_size = min_8bit_size
        self._dev = None
        self._rates = None       # learning rates that lr_dev holds
        self._ws = None
        self._held = []
        self._restored_step = None
        self.grad_norm = None    # device scalar: total gradient norm of the last clipped step, before clipping

    def add_param_group(self, group):
        if len(self.param_groups) >= _ffi.ADAMW_MAX_GROUPS:
            raise ValueError(f"FusedAdamW takes up to {_ffi.ADAMW_MAX_GROUPS} parameter groups")
        params = group["params"]
        if not torch.is_tensor(params) and not isinstance(params, set):
            params = list(params)
            # (a parameter given twice would be updated by two workgroups at once)
            if len({id(p[1] if isinstance(p, tuple) else p) for p in params}) != len(params):
                raise ValueError("FusedAdamW: a parameter appears twice in a group")
            group = {**group, "params": params}
        self._check_group({**self.defaults, **group})
        super().add_param_group(group)

    @staticmethod
    def _check_group(g):
        b1, b2 = g["betas"]
        if not (0 <= b1 < 1 and 0 <= b2 < 1 and g["eps"] >= 0 and g["weight_decay"] >= 0 and g["lr"] >= 0):
            raise ValueError("FusedAdamW: betas in [0, 1), eps, weight_decay and lr not negative")
        for other in ("amsgrad", "maximize"):
            if g.get(other):
                raise ValueError(f"FusedAdamW: {other} is not built")

    def __getstate__(self):
        steps = int(self.step_count.item()) if self._dev is not None else self._restored_step
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "state_bits": self.state_bits,
                "min_8bit_size": self.min_8bit_size, "_restored_step": steps}

    def __setstate__(self, state):
        super().__setstate__(state)
        if "_dev" not in self.__dict__:      # a copy or an unpickled optimizer: device scalars are made anew
            self._dev = self._rates = self._ws = self.grad_norm = None
            self._held = []

    def _is8(self, p):
        return self.state_bits == 8 and p.numel() >= self.min_8bit_size

    def _init_device(self, dev):
        self._dev = dev
        if self._restored_step is None:
            self._restored_step = max((int(st["step"]) for st in self.state.values() if "step" in st), default=0)
        self.step_count = torch.full((1,), self._restored_step, dtype=torch.int64, device=dev)
        self.lr_dev = torch.zeros(_ffi.ADAMW_MAX_GROUPS, dtype=torch.float32, device=dev)
        self.grad_norm = torch.zeros(1, dtype=torch.float32, device=dev)
        tensors = sum(len(g["params"]) for g in self.param_groups)
        self._ws = torch.empty(_ffi.load().rk_adamw_ws_bytes(tensors) // 8, dtype=torch.float64, device=dev)

    def _refuse(self, p, g):
        if not p.is_cuda:
            raise _ffi.RkError(_ffi.RK_ERR_NODEV, "FusedAdamW: parameters on a HIP device only")
        if p.device != self._dev or g.device != self._dev:
            raise _ffi.RkError(_ffi.RK_ERR_UNSUPPORTED, f"FusedAdamW: all parameters on one device ({self._dev})")
        raise _ffi.RkError(_ffi.RK_ERR_UNSUPPORTED, "FusedAdamW: contiguous fp32, bfloat16 or fp16 parameters on a HIP "
                           "device with dense gradients of their type or fp32 only")

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._dev is None:
            first = next((p for g in self.param_groups for p in g["params"] if p.grad is not None and p.numel()), None)
            if first is None:
                return loss
            if not first.is_cuda:
                self._refuse(first, first.grad)
            _not_in_a_capture()
            self._init_device(first.device)
        self.sync_lr()
        need = self._launch()
        if need:
            _not_in_a_capture()
            self._held.append(self._ws)      # a recorded step goes on with the one that it was recorded with
            self._ws = torch.empty(need // 8, dtype=torch.float64, device=self._dev)
            self._launch()
        return loss

    def _launch(self):
        # (moments that a capture made would start from zero at every replay)
        return _ffi.torch_ops().adamw_step(self.param_groups, self.state,
                                           self.min_8bit_size if self.state_bits == 8 else _NEVER, _not_in_a_capture,
                                           self._refuse, self.step_count, self.lr_dev, self.max_grad_norm or 0.0,
                                           self.grad_norm, self._ws)

    def sync_lr(self):
        """Push learning rates changed by a scheduler to device memory.  step() does it, and so do the recorded steps
        of train_step and dist_train; call it before replaying a graph of your own, outside the capture."""
        rates = [float(g["lr"]) for g in self.param_groups]
        if self._dev is None or rates == self._rates:
            return
        if torch.cuda.is_current_stream_capturing():
            if self._rates is None:
                raise RuntimeError("run one optimizer step before capturing it in a graph")
            return
        for k, rate in enumerate(rates):
            if self._rates is None or k >= len(self._rates) or self._rates[k] != rate:
                self.lr_dev[k].fill_(rate)
        self._rates = rates

    def state_dict(self):
        """torch.optim.AdamW's layout (and the keys of 8-bit moments): every parameter's state carries `step`
        beside its moments (reading the device counter synchronises)."""
        if self._dev is not None:
            t = float(self.step_count.item())
            for st in self.state.values():
                if st:
                    st["step"] = torch.tensor(t)
        return super().state_dict()

    def _entries(self, state_dict):
        """{parameter: its moments in the checkpoint}, checked: nothing is replaced by a checkpoint of other sizes."""
        for g in state_dict["param_groups"]:
            self._check_group({**self.defaults, **g})
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return {}                                # (another model's: torch says so)
        entries = {}
        for i, p in zip([i for g in groups for i in g["params"]], [p for g in self.param_groups for p in g["params"]]):
            src = saved.get(i)
            if not src or not ("exp_avg" in src or "exp_avg8" in src):
                continue
            n, blocks = p.numel(), -(-p.numel() // _ffi.ADAMW_BLOCK)
            sizes = ((n, n) if "exp_avg" in src else
                     (blocks * _ffi.ADAMW_BLOCK, blocks, blocks * _ffi.ADAMW_BLOCK, blocks))
            for k, size in zip(_STATE32 if "exp_avg" in src else _STATE8, sizes):
                if not torch.is_tensor(src.get(k)) or src[k].numel() != size:
                    raise ValueError(f"FusedAdamW: {k} of a checkpoint does not fit a parameter of {tuple(p.shape)}")
            entries[p] = src
        return entries

    def _moments_of(self, p, src):
        """A parameter's state from a checkpoint's, in the form this optimizer holds it."""
        src = {k: v.to(p.device) if torch.is_tensor(v) else v for k, v in src.items()}
        st = {"step": torch.tensor(float(src.get("step", 0)))}
        if self._is8(p) and "exp_avg8" in src:
            st.update({k: src[k].clone() for k in _STATE8})
        elif self._is8(p):
            st["exp_avg8"], st["exp_avg8_scale"] = encode_moment(src["exp_avg"])
            st["exp_avg_sq8"], st["exp_avg_sq8_scale"] = encode_moment(src["exp_avg_sq"].float().sqrt(), True)
        elif "exp_avg" in src:
            st.update({k: src[k].detach().float().reshape(p.shape).clone() for k in _STATE32})
        else:
            st["exp_avg"] = decode_moment(src["exp_avg8"], src["exp_avg8_scale"], p)
            st["exp_avg_sq"] = decode_moment(src["exp_avg_sq8"], src["exp_avg_sq8_scale"], p).square()
        return st

    def load_state_dict(self, state_dict):
        """Moments and step count of a checkpoint: this optimizer's with either number of bits, or
        torch.optim.AdamW's.  Moments are converted to the form this optimizer holds.  Buffers that exist
        keep their memory and take the checkpoint's values (zeros, where it has no moments of their parameter:
        one saved before the first step has none), so a step recorded in a HIP graph before the load goes on
        with them.  Buffers of another form than the checkpoint's become are not used again, and not freed
        either.  Call it outside graph capture."""
        old = {p: {k: v for k, v in st.items() if k != "step" and torch.is_tensor(v)} for p, st in self.state.items()}
        entries = self._entries(state_dict)
        # (torch would cast floating state to the parameter's type, all of it at once: the groups are its part, the
        # moments are taken from the checkpoint itself, a parameter at a time)
        super().load_state_dict({**state_dict, "state": {}})
        for p, held in old.items():
            if held:
                self.state[p] = dict(held)
        for p, src in entries.items():
            st, held = self._moments_of(p, src), old.pop(p, {})
            for k, v in st.items():
                have = held.get(k)
                if have is not None and have.shape == v.shape and have.dtype == v.dtype:
                    have.copy_(v)
                    st[k] = held.pop(k)
            self._held += held.values()
            self.state[p] = st
        for held in old.values():
            for v in held.values():
                (v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v).zero_()
        self._restored_step = max((int(st["step"]) for st in self.state.values() if "step" in st), default=0)
        if self._dev is not None:
            self.step_count.fill_(self._restored_step)
            self._rates = None
            self.sync_lr()
