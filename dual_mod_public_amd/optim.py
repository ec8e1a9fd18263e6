"""AdamW over all tensors of a model in one launch (dm_adamw_step_counted), with 32-bit or 8-bit states and clipping by the
global gradient norm.

    opt = trunk.optimizer(lr=3e-4, weight_decay=0.1, max_norm=1.0)      # or AdamW(params, grads=..., ...)
    trunk.train_step(idx, targets)
    opt.step()
    trunk.refresh()

Parameters are the framework's fp32 masters. Gradients are fixed buffers given once (``grads``: fp32 or bf16, as
HipTrunk's views of its flat buffer) or, without them, the parameters' ``.grad`` at each step: a parameter without one is
left as it is, its states too, and its bias corrections count the steps that it took part in. Everything a step
changes beside the parameters lives on the device (``lr``, ``steps``, ``tensor_steps``, ``norm``, ``skipped``), so a step
can be captured into a HIP graph and replayed. A replay works on the parameters and gradients that the step was captured
with, which the optimizer keeps allocated from then on (keep the optimizer as long as the graph), and does not tell torch
that the parameters changed: call ``mark_updated()`` after it where something watches their versions (GraphDecoder,
SwiGLU.decode).

A step whose tensors lie where they lay before is launches alone. One that finds a tensor moved writes the launch plan again,
which waits for the device: let ``.grad`` stay (``zero_grad(set_to_none=False)``) or give ``grads`` where steps are short.

8-bit states hold a byte per element and moment, and a byte per 256 elements and moment: blocks with a power-of-two
scale, four significant bits per element, rounded stochastically by a hash of seed, step and element, so runs repeat
bit for bit. A NaN or infinity in a state makes its block NaN; ``skip_nonfinite`` leaves such steps out.
"""

import ctypes
from bisect import bisect_left
from itertools import chain

import torch

from . import _lib as L


class AdamW:
    """params: tensors, or dicts ``{"params": [...], "weight_decay": x, "lr_scale": x}``. grads: as many buffers in the
    same order (see above). lr: the learning rate (``set_lr`` changes it). max_norm: clip by the global norm (None: no
    clipping). state_bits: 32 or 8. seed: of the 8-bit states' rounding."""

    def __init__(self, params, grads=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_norm=None,
                 skip_nonfinite=False, state_bits=32, seed=0):
        groups = [dict(g) if isinstance(g, dict) else {"params": g} for g in params]
        for g in groups:
            if "params" not in g or set(g) - {"params", "weight_decay", "lr_scale"}:
                raise ValueError(f"parameter group of {sorted(g)}")
            g["params"] = [g["params"]] if torch.is_tensor(g["params"]) else list(g["params"])
        self.params = [p for g in groups for p in g["params"]]
        self._decay = [float(g.get("weight_decay", weight_decay)) for g in groups for _ in g["params"]]
        self._scale = [float(g.get("lr_scale", 1.0)) for g in groups for _ in g["params"]]
        if not self.params:
            raise ValueError("no parameters")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits={state_bits} (32 or 8)")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and 2.0 ** -126 <= eps < 2.0 ** 128):
            raise ValueError(f"betas={betas} eps={eps} (eps a normal fp32 number)")
        if max_norm is not None and not 0 < max_norm < float("inf"):
            raise ValueError(f"max_norm={max_norm}")
        self.device = self.params[0].device
        for i, p in enumerate(self.params):
            if not p.is_cuda or p.device != self.device or p.dtype != torch.float32 or not p.is_contiguous():
                raise ValueError(f"parameter {i}: {p.dtype} {tuple(p.shape)} on {p.device}; contiguous fp32 on one GPU")
        spans = sorted((p.data_ptr(), p.data_ptr() + 4 * p.numel()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory")
        starts = [a for a, _ in spans]
        self.grads = None
        if grads is not None:
            self.grads = list(grads)
            if len(self.grads) != len(self.params):
                raise ValueError(f"{len(self.grads)} gradients for {len(self.params)} parameters")
            for i, (p, g) in enumerate(zip(self.params, self.grads)):
                self._check_grad(i, p, g)
                k = bisect_left(starts, g.data_ptr() + g.numel() * g.element_size())   # parameters that start before its end
                if k and g.numel() and spans[k - 1][1] > g.data_ptr():
                    raise ValueError(f"gradient {i} shares memory with a parameter")
        self.betas, self.eps, self.max_norm = (float(betas[0]), float(betas[1])), float(eps), max_norm
        self.skip_nonfinite, self.state_bits, self.seed = bool(skip_nonfinite), state_bits, int(seed) & 0xffffffff

        # flat states: tensor i's elements from block ``_block0[i]`` on
        self._block0, n = [], 0
        self._sizes = [p.numel() for p in self.params]
        for p in self.params:
            self._block0.append(n)
            n += -(-p.numel() // L.DM_ADAMW_BLOCK)
        self.n_blocks = n
        kw = dict(device=self.device)
        dt = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg, self.exp_avg_sq = (torch.zeros(n * L.DM_ADAMW_BLOCK, dtype=dt, **kw) for _ in range(2))
        self.exp_avg_exponent = self.exp_avg_sq_exponent = None
        if state_bits == 8:
            self.exp_avg_exponent, self.exp_avg_sq_exponent = (torch.ones(n, dtype=torch.uint8, **kw) for _ in range(2))
        self.lr = torch.full((), float(lr), dtype=torch.float32, **kw)
        self.steps = torch.zeros((), dtype=torch.int64, **kw)        # steps taken
        self.norm = torch.zeros((), dtype=torch.float32, **kw)       # the last step's gradient norm (before clipping)
        self.skipped = torch.zeros((), dtype=torch.int32, **kw)      # steps left out by skip_nonfinite
        self.tensor_steps = torch.zeros(len(self.params), dtype=torch.int64, **kw)   # steps with a gradient, per parameter
        self._ws = torch.empty(L.DM_ADAMW_WORKSPACE + 8 * len(self.params), dtype=torch.uint8, **kw)
        self._key = self._plan = self._a = None
        self._in_graphs, self._graphs_hold = [], []    # plans that captured steps read, and what those read and write
        torch.cuda.current_stream(self.device).synchronize()   # the buffers are ready on every stream

    def _check_grad(self, i, p, g):
        if g.shape != p.shape or g.device != p.device or not g.is_contiguous():
            raise ValueError(f"gradient {i}: {tuple(g.shape)} on {g.device}; contiguous {tuple(p.shape)} on {p.device}")
        L.dtype_code(g.dtype)

    def _args(self):
        """dm_adamw_args of a step now; the plan is written again where a tensor has moved."""
        grads = self.grads if self.grads is not None else [p.grad for p in self.params]
        key = [None if t is None else t.data_ptr() for t in chain(self.params, grads)]
        if self.grads is None:   # a new .grad may have an old one's address
            key += [None if g is None else (g.dtype, g.is_contiguous(), g.numel()) for g in grads]
        if key != self._key:
            self._write_plan(grads)
            self._key = key
        if torch.cuda.is_current_stream_capturing() and not any(self._plan is t for t in self._in_graphs):
            self._in_graphs.append(self._plan)
            self._graphs_hold.append((self._held, [g.detach() for g in grads if g is not None]))
        return self._a

    def _write_plan(self, grads):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a tensor has moved since the last step; take one step before capturing")
        self._key = None
        rows = []
        for i, (p, g) in enumerate(zip(self.params, grads)):
            if p.numel() != self._sizes[i]:   # its states have their place between the others'
                raise ValueError(f"parameter {i} now has {p.numel()} elements; its states were made for {self._sizes[i]}")
            if g is None or p.numel() == 0:   # its place in tensor_steps
                rows.append(L.dm_adamw_tensor(None, None, 0, 0, 0.0, 0.0, L.DM_F32, 0))
                continue
            self._check_grad(i, p, g)
            if p.dtype != torch.float32 or p.device != self.device or not p.is_contiguous():
                raise ValueError(f"parameter {i} is now {p.dtype} on {p.device}")
            rows.append(L.dm_adamw_tensor(p.data_ptr(), g.data_ptr(), p.numel(), self._block0[i], self._decay[i],
                                          self._scale[i], L.dtype_code(g.dtype), 0))
        if not any(t.n for t in rows):
            raise ValueError("no parameter has a gradient")
        arr = (L.dm_adamw_tensor * len(rows))(*rows)
        nb = L.lib().dm_adamw_plan_bytes(arr, len(rows))
        if nb == 0:
            raise L.DMError("dm_adamw_plan_bytes: " + L.lib().dm_last_error().decode())
        host, n = torch.empty(nb, dtype=torch.uint8), ctypes.c_int64()
        L.check(L.lib().dm_adamw_plan(arr, len(rows), host.data_ptr(), nb, ctypes.byref(n)))
        self._held = [p.detach() for p in self.params]   # what the plan writes stays allocated
        torch.cuda.synchronize(self.device)   # no step still reads the plan that this one replaces
        self._plan = host.to(self.device)
        torch.cuda.current_stream(self.device).synchronize()
        a = self._a = L.dm_adamw_args()
        a.plan, a.n_chunks, a.n_tensors, a.state_bits = self._plan.data_ptr(), n.value, len(rows), self.state_bits
        a.exp_avg, a.exp_avg_sq = self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr()
        a.exp_avg_exponent, a.exp_avg_sq_exponent = L.ptr(self.exp_avg_exponent), L.ptr(self.exp_avg_sq_exponent)
        a.beta1, a.beta2, a.eps = self.betas[0], self.betas[1], self.eps
        a.max_norm, a.skip_nonfinite, a.seed = self.max_norm or 0.0, int(self.skip_nonfinite), self.seed
        a.lr, a.steps = self.lr.data_ptr(), self.steps.data_ptr()
        a.norm, a.skipped = self.norm.data_ptr(), self.skipped.data_ptr()
        a.workspace, a.workspace_bytes = self._ws.data_ptr(), self._ws.numel()

    def _call(self, fn):
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._call(fn)
        L.call_on(self.device, fn, L.byref(self._args()))

    def _counted(self, args, stream):
        return L.lib().dm_adamw_step_counted(args, self.tensor_steps.data_ptr(), stream)

    def step(self):
        """One step. Returns the gradients' global norm before clipping (a device scalar, overwritten by the next
        step) where it is computed: with max_norm or skip_nonfinite; else None."""
        self._call(self._counted)
        self.mark_updated()
        return self.norm if self.max_norm is not None or self.skip_nonfinite else None

    def grad_norm(self):
        """The gradients' global norm alone (a device scalar, overwritten by the next call or step)."""
        self._call(L.lib().dm_grad_norm)
        return self.norm

    def mark_updated(self):
        """Tell torch that the parameters were written (their version counters): done by ``step``, needed after the
        replay of a captured one."""
        torch.autograd.graph.increment_version(self.params)

    def set_lr(self, lr):
        self.lr.fill_(float(lr))

    def views(self, flat):
        """A flat state (``exp_avg``, one of ``state_values()``) as one tensor per parameter, in its shape."""
        o = [b * L.DM_ADAMW_BLOCK for b in self._block0]
        return [flat[k:k + p.numel()].view(p.shape) for k, p in zip(o, self.params)]

    def state_values(self):
        """(first, second) moments as flat tensors of numbers: the fp32 states, or the 8-bit states' values in bf16
        (exact)."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        out = [torch.empty(self.exp_avg.numel(), device=self.device, dtype=torch.bfloat16) for _ in range(2)]
        with torch.cuda.device(self.device):
            for second, (c, e) in enumerate(((self.exp_avg, self.exp_avg_exponent), (self.exp_avg_sq, self.exp_avg_sq_exponent))):
                L.check(L.lib().dm_adamw_values(c.data_ptr(), e.data_ptr(), self.n_blocks, second, out[second].data_ptr(),
                                                L.stream_ptr()))
        return tuple(out)

    def state_dict(self):
        """The states (the live tensors, as torch's modules give theirs), the parameters' sizes, the step counts, the
        learning rate and, of 8-bit states, the seed of their rounding."""
        d = dict(steps=int(self.steps), lr=float(self.lr), state_bits=self.state_bits, sizes=list(self._sizes), exp_avg=self.exp_avg,
                 exp_avg_sq=self.exp_avg_sq, tensor_steps=self.tensor_steps)
        if self.state_bits == 8:
            d.update(seed=self.seed, exp_avg_exponent=self.exp_avg_exponent, exp_avg_sq_exponent=self.exp_avg_sq_exponent)
        return d

    @torch.no_grad()
    def load_state_dict(self, d):
        """Copies state_dict()'s values in; the learning rate and the seed only where they are given (a step captured before
        keeps its seed). Without ``tensor_steps`` every parameter counts as one that took part in all steps."""
        if d["state_bits"] != self.state_bits:
            raise ValueError(f"states of {d['state_bits']} bits for an optimizer of {self.state_bits}")
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exponent", "exp_avg_sq_exponent"] if self.state_bits == 8 else [])
        for n in names:
            t = getattr(self, n)
            if d[n].shape != t.shape or d[n].dtype != t.dtype:
                raise ValueError(f"{n}: {d[n].dtype} {tuple(d[n].shape)}, {t.dtype} {tuple(t.shape)} is needed")
        if list(d.get("sizes", self._sizes)) != self._sizes:
            raise ValueError("states of parameters of other sizes or in another order")
        counts = d.get("tensor_steps")
        if counts is not None and tuple(counts.shape) != (len(self.params),):
            raise ValueError(f"tensor_steps: {tuple(counts.shape)}, one per parameter ({len(self.params)}) is needed")
        for n in names:
            getattr(self, n).copy_(d[n])
        self.steps.fill_(int(d["steps"]))
        if counts is None:
            self.tensor_steps.fill_(int(d["steps"]))
        else:
            self.tensor_steps.copy_(counts)
        if "lr" in d:
            self.set_lr(d["lr"])
        if "seed" in d:
            self.seed = int(d["seed"]) & 0xffffffff
            if self._a is not None:
                self._a.seed = self.seed
