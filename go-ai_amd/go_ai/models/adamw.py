"""AdamW over many tensors in one launch (goai_adamw_*), with the moments in 32 or in 8 bits."""
import ctypes
import math

import torch

BLOCK = 256          # elements that share one scale of an 8-bit moment

_dtype_of, _shape_of = torch.Tensor.dtype.__get__, torch.Tensor.shape.__get__
_device_of, _is_contiguous, _address_of = torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _ctypes_table(ctype, values):
    return (ctype * max(len(values), 1))(*values)


class AdamW:
    """torch.optim.AdamW's update over a list of GPU tensors:

        g = gradient * min(1, max_norm / |all gradients|)      (max_norm = 0: as it is)
        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    params: contiguous tensors of one GPU (float32, bfloat16 or float16, in any mixture), or None / host tensors (what
    RLNet.parameters() yields): then the optimiser belongs to the net that it is first handed to (RLNet.optimize,
    RLNet.train_step), which gives it its parameters.  weight_decay and grad_dtype (None: each parameter's own type) are one value or
    one per tensor.  state_bits = 8 holds the moments in a byte each, in blocks of 256 elements with a scale; from the 17th step after they
    were set on they are rounded at random, so that changes below half a code add up (sqrt(v) scatters by about 0.15 of itself,
    its mean follows float32's); the same steps give the same bits.

    step(grads) takes the gradients as a list in the parameters' order (None: that tensor stays as it is).  With max_norm a norm
    that is not finite skips the step: parameters and moments stay as they are, and it is not counted; `norm` is the last step's
    norm (a GPU scalar).

    A step can be captured into a graph: step(grads, captured=True) reads lr and the bias corrections from GPU memory when it
    runs; call advance() before the capture's first replay and before every further one, on the stream that replays."""

    def __init__(self, params=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=0.0,
                 grad_dtype=None, ctx=None):
        self.lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.weight_decay, self.state_bits, self.max_norm, self.grad_dtype = weight_decay, int(state_bits), float(max_norm), grad_dtype
        if not (0.0 <= self.lr < math.inf and all(0.0 <= b < 1.0 for b in self.betas) and 1e-30 <= self.eps < math.inf):
            raise ValueError("AdamW: lr >= 0, betas in [0, 1), eps >= 1e-30")
        if self.state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits must be 8 or 32")
        if not 0.0 <= self.max_norm:
            raise ValueError("AdamW: max_norm must not be negative")
        self._calls = 0                                          # steps, skipped ones among them
        self.params = None
        self._h = self._ctx = self._net = self._held = None
        params = None if params is None else list(params)
        if params and all(torch.is_tensor(p) and p.is_cuda for p in params):
            self.bind(params, ctx)
        elif params and any(torch.is_tensor(p) and p.is_cuda for p in params):
            raise ValueError("AdamW: parameters on the GPU and on the host")

    def zero_grad(self):
        pass

    # ---- parameters --------------------------------------------------------------------------
    def bind(self, params, ctx=None):
        """Take these GPU tensors as the parameters; fresh moments, or those that load_state_dict left for them."""
        from .. import _hip
        from ..engine import ELEM_TYPES, Context
        params = list(params)
        n = len(params)
        if not n:
            raise ValueError("AdamW: no parameters")
        device = params[0].device
        if ctx is not None and ctx.device != device:
            raise ValueError(f"AdamW: parameters on {device}, a context of {ctx.device}")
        for p in params:
            if not p.is_cuda or p.device != device or p.dtype not in ELEM_TYPES or not p.is_contiguous():
                raise ValueError("AdamW: parameters are contiguous float32, bfloat16 or float16 tensors of one GPU, got "
                                 f"{p.dtype} on {p.device}, strides {p.stride()}")

        def each(x, what):
            x = list(x) if isinstance(x, (list, tuple)) else [x] * n
            if len(x) != n:
                raise ValueError(f"AdamW: {n} parameters, {len(x)} values of {what}")
            return x
        decays = [float(d) for d in each(self.weight_decay, "weight_decay")]
        gtypes = [p.dtype if g is None else g for p, g in zip(params, each(self.grad_dtype, "grad_dtype"))]
        if any(g not in ELEM_TYPES for g in gtypes):
            raise ValueError("AdamW: gradients are float32, bfloat16 or float16")
        numels = _ctypes_table(ctypes.c_int64, [p.numel() for p in params])
        elems = _hip.lib.goai_adamw_state_elems(n, numels)
        state = torch.uint8 if self.state_bits == 8 else torch.float32
        blocks = max(elems, 1) // BLOCK if self.state_bits == 8 else 0
        m, v = [torch.zeros(elems, dtype=state, device=device) for _ in range(2)]
        scales = torch.zeros((2, max(blocks, 1)), dtype=torch.float32, device=device)
        held = self._held
        if held is not None:
            self._check_moments(held["exp_avg"], held["exp_avg_sq"], [p.shape for p in params], "the loaded state's")
        ctx = ctx if ctx is not None else Context(9, device.index)
        ctx._bind()
        h = ctypes.c_void_p()
        eight = self.state_bits == 8
        _hip.check(_hip.lib.goai_adamw_init(
            ctx._h, n, _ctypes_table(ctypes.c_void_p, [p.data_ptr() for p in params]),
            _ctypes_table(ctypes.c_int32, [ELEM_TYPES[p.dtype] for p in params]), _ctypes_table(ctypes.c_int32, [ELEM_TYPES[g] for g in gtypes]),
            numels, _ctypes_table(ctypes.c_float, decays), self.state_bits, m.data_ptr() or scales.data_ptr(), v.data_ptr() or scales.data_ptr(),
            scales[0].data_ptr() if eight else None, scales[1].data_ptr() if eight else None, ctypes.byref(h)))
        self.close()                                             # (a refused bind leaves the optimiser as it was)
        self._h, self._ctx, self._held = h, ctx, None
        self.params, self.device, self._net = params, device, None
        self._addresses = [p.data_ptr() for p in params]
        # autograd's counters of changes in place (views share their base's): a graph that saved a parameter before a step says so
        bases = [p if p._base is None else p._base for p in params]
        self._versions = list({id(b): b for b in bases}.values())
        self._gtypes, self._shapes, self._devices = gtypes, [p.shape for p in params], [device.index] * n
        self._m, self._v, self._scales, self._elems = m, v, scales, elems
        self._table = _ctypes_table(ctypes.c_void_p, [None] * n)
        self._clip = torch.zeros(2, dtype=torch.float32, device=device)
        self._scalars = None
        self.offsets, at = [], 0
        for p in params:
            self.offsets.append(at)
            at += -(-p.numel() // BLOCK) * BLOCK
        self._calls = 0
        if held is not None:
            self._load(held)
        return self

    def close(self):
        if self._h is not None:
            from .. import _hip
            _hip.lib.goai_adamw_destroy(None if self._ctx.closed else self._ctx._h, self._h)
        self._h = None

    def __getstate__(self):
        if self._h is not None:
            raise TypeError("AdamW: moments on the GPU are not copied or pickled; use state_dict")
        return self.__dict__

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _bound(self):
        if self._h is None:
            raise RuntimeError("AdamW: no parameters yet: give it GPU tensors, or hand it to a net's train_step / optimize")
        self._ctx._bind()

    # ---- the step ----------------------------------------------------------------------------
    @property
    def steps(self):
        """The number of steps behind the moments.  With max_norm this waits for the GPU, which knows the skipped ones."""
        if self._h is None:
            return self._held["steps"] if self._held is not None else self._calls
        from .. import _hip
        skipped = ctypes.c_int64()
        if not self._ctx.closed:
            self._ctx._bind()
        _hip.check(_hip.lib.goai_adamw_skipped(None if self._ctx.closed else self._ctx._h, self._h, ctypes.byref(skipped)))
        return self._calls - skipped.value

    def _grads(self, grads):
        if list(map(_address_of, self.params)) != self._addresses:
            raise RuntimeError("AdamW: a parameter's memory was replaced since bind(): bind the optimiser again (fresh moments)")
        if len(grads) != len(self.params):
            raise ValueError(f"AdamW: {len(self.params)} parameters, {len(grads)} gradients")
        try:                                                     # one pass per property: a third faster than tensor by tensor
            if (list(map(_dtype_of, grads)) == self._gtypes and list(map(_shape_of, grads)) == self._shapes
                    and list(map(_device_of, grads)) == self._devices and all(map(_is_contiguous, grads))):
                self._table[:] = list(map(_address_of, grads))
                return self._table
        except TypeError:                                        # a gradient that is None
            pass
        table = self._table
        for i, (g, dtype, shape) in enumerate(zip(grads, self._gtypes, self._shapes)):
            if g is None:
                table[i] = None
            elif torch.is_tensor(g) and g.dtype is dtype and g.shape == shape and g.device == self.device and g.is_contiguous():
                table[i] = g.data_ptr()
            else:
                what = f"{g.dtype} of shape {tuple(g.shape)} on {g.device}, strides {g.stride()}" if torch.is_tensor(g) else type(g).__name__
                raise ValueError(f"AdamW: gradient {i} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {self.device}, got {what}")
        return table

    def advance(self):
        """The next step's number; writes lr and the bias corrections of that step where a captured step reads them."""
        from .. import _hip
        self._bound()
        if self._scalars is None:
            self._scalars = torch.zeros(3, dtype=torch.float64, device=self.device)
        _hip.check(_hip.lib.goai_adamw_scalars(self._ctx._h, self._h, self._calls + 1, float(self.lr), self.betas[0], self.betas[1],
                                               self._scalars.data_ptr()))
        self._calls += 1

    def step(self, grads, captured=False):
        """One step on the current stream: number `steps` + 1 (captured: see advance)."""
        from .. import _hip
        self._bound()
        table = self._grads(grads)
        if captured and self._scalars is None:
            raise RuntimeError("AdamW: call advance() before a captured step")
        torch.autograd.graph.increment_version(self._versions)
        t = self._calls if captured else self._calls + 1
        _hip.check(_hip.lib.goai_adamw_step(self._ctx._h, self._h, table, max(t, 1), float(self.lr), self.betas[0], self.betas[1], self.eps,
                                            self.max_norm, self._clip.data_ptr() if self.max_norm else None,
                                            self._scalars.data_ptr() if captured else None))
        self._calls = t

    @property
    def norm(self):
        """The gradients' global norm at the last step with max_norm (before clipping): a GPU scalar."""
        return self._clip[0]

    def grad_norm(self, grads):
        """The global norm of these gradients (a GPU scalar), without a step: what a step with max_norm would clip."""
        from .. import _hip
        self._bound()
        out = torch.empty(2, dtype=torch.float32, device=self.device)
        _hip.check(_hip.lib.goai_adamw_grad_norm(self._ctx._h, self._h, self._grads(grads), math.inf, out.data_ptr()))
        return out[0]

    # ---- moments -----------------------------------------------------------------------------
    def moments(self):
        """(exp_avg, exp_avg_sq) as flat float32 GPU tensors: tensor i's at [offsets[i] : offsets[i] + numel].  The optimiser's own
        buffers for state_bits = 32, the values that the codes stand for (new tensors) for 8."""
        self._bound()
        if self.state_bits == 32:
            return self._m, self._v
        from .. import _hip
        m, v = [torch.empty(self._elems, dtype=torch.float32, device=self.device) for _ in range(2)]
        if self._elems:
            _hip.check(_hip.lib.goai_adamw_moments(self._ctx._h, self._h, m.data_ptr(), v.data_ptr()))
        return m, v

    def _carry(self, state=None):
        """The moments as they are held, and the step number: out of here, or (to the same parameters in other memory) back in."""
        self._bound()
        if state is None:
            return self.steps, self._m, self._v, self._scales
        for mine, theirs in zip((self._m, self._v, self._scales), state[1:]):
            mine.copy_(theirs)
        self._calls = state[0]

    def _split(self, flat):
        return [flat[a:a + p.numel()].view(p.shape) for a, p in zip(self.offsets, self.params)]

    @staticmethod
    def _check_moments(exp_avg, exp_avg_sq, shapes, what):
        if len(exp_avg) != len(shapes) or len(exp_avg_sq) != len(shapes):
            raise ValueError(f"AdamW: {len(shapes)} parameters, {what} for {len(exp_avg)} and {len(exp_avg_sq)}")
        for a, b, s in zip(exp_avg, exp_avg_sq, shapes):
            if a.shape != s or b.shape != s:
                raise ValueError(f"AdamW: a parameter of shape {tuple(s)}, {what} of shapes {tuple(a.shape)} and {tuple(b.shape)}")

    def load_moments(self, exp_avg, exp_avg_sq, steps):
        """Continue from these moments (one float tensor per parameter) after `steps` steps; 8-bit moments are rounded to their codes."""
        self._bound()
        if int(steps) < 0:
            raise ValueError("AdamW: steps must not be negative")
        self._check_moments(exp_avg, exp_avg_sq, self._shapes, "moments")
        from .. import _hip
        tables, held = [], []
        for given in (exp_avg, exp_avg_sq):
            given = [x if x.dtype is torch.float32 and x.device == self.device and x.is_contiguous()
                     else x.to(self.device, dtype=torch.float32).contiguous() for x in given]
            held.append(given)
            tables.append(_ctypes_table(ctypes.c_void_p, list(map(_address_of, given))))
        _hip.check(_hip.lib.goai_adamw_load_moments(self._ctx._h, self._h, *tables))
        self._calls = int(steps)

    def state_dict(self):
        """steps and the moments as float32 host tensors in the parameters' order, with the parameters' names if they are a net's; for
        state_bits = 8 with their codes and scales too, which the values alone give back to some roundings only."""
        if self._h is None and self._held is not None:
            return dict(self._held)
        m, v = self.moments()
        state = {"steps": self.steps, "exp_avg": [x.cpu().clone() for x in self._split(m)], "exp_avg_sq": [x.cpu().clone() for x in self._split(v)]}
        if self.state_bits == 8:
            state["codes"] = [[x.cpu().clone() for x in views] for views in self._codes()]
        if self._net is not None:
            state["names"] = list(self._net_names)
        return state

    def _codes(self):
        """Views of the 8-bit moments' buffers by tensor: codes and scales of the first, codes and scales of the second."""
        blocks = [(a // BLOCK, -(-p.numel() // BLOCK)) for a, p in zip(self.offsets, self.params)]
        return [views for flat, scales in ((self._m, self._scales[0]), (self._v, self._scales[1]))
                for views in ([flat[a:a + p.numel()] for a, p in zip(self.offsets, self.params)], [scales[a:a + n] for a, n in blocks])]

    def load_state_dict(self, state):
        """Continue from a state_dict.  An optimiser that has no parameters yet keeps it for those that it is bound to: a net's AdamW
        is resumed by loading its state before the net's next train_step, optimize or policy_step."""
        if int(state["steps"]) < 0:
            raise ValueError("AdamW: steps must not be negative")
        if self._h is None:
            self._held = {**state, "steps": int(state["steps"])}
            return
        if self._net is not None:
            state = self._in_order(state, self._net_names)
        self._load(state)

    def _load(self, state):
        self.load_moments(state["exp_avg"], state["exp_avg_sq"], state["steps"])
        if self.state_bits == 8 and "codes" in state:
            for mine, theirs in zip(self._codes(), state["codes"]):
                for a, b in zip(mine, theirs):
                    a.copy_(b)
            # values that were changed since they were saved count, not the codes beside them
            for mine, theirs in zip(self.moments(), (state["exp_avg"], state["exp_avg_sq"])):
                if not all(torch.equal(a, b.to(self.device, dtype=torch.float32)) for a, b in zip(self._split(mine), theirs)):
                    return self.load_moments(state["exp_avg"], state["exp_avg_sq"], state["steps"])

    @staticmethod
    def _in_order(state, names):
        """A net's state in the order of `names`."""
        if "names" not in state or list(state["names"]) == list(names):
            return state
        if sorted(state["names"]) != sorted(names):
            raise ValueError("AdamW: the loaded state is of another net's parameters")
        at = [list(state["names"]).index(k) for k in names]
        turned = {**state, "names": list(names), **{k: [state[k][i] for i in at] for k in ("exp_avg", "exp_avg_sq")}}
        if "codes" in state:
            turned["codes"] = [[views[i] for i in at] for views in state["codes"]]
        return turned
