"""Gradient clipping + AdamW with the moments in 8 bits (``mmt_clip_adamw8_step``, csrc/clip_adamw8.hip): ``ClipAdamW8`` beside
``optim.ClipAdamW``.  The optimizer state of a parameter is 2.06 bytes an element instead of 8, and a step moves 16 bytes an element
instead of 28.  Tensors of fewer than ``min_8bit_size`` elements keep 32-bit moments; both kinds are stepped by the same launch.

Further than ClipAdamW it takes bf16 parameters (rounded stochastically: no fp32 copy is needed for small updates to count), several
parameter groups under one clipping norm, and parameters that join later (every one has its own step count).
"""
import itertools
import math
import operator

import numpy as np
import torch
from torch._C._dynamo.guards import TensorGuards

from .. import _lib
from .optim import RING, _dense
from .optim import _same_layout as _same_order

BLOCK = 32          # elements that share a scale byte
ALIGN = 256         # every tensor's moments begin at a multiple of this many elements of the state buffers
COLUMNS = 9         # MMT_ADAMW8_COLUMNS
_GRAD, _ADDRESS, _NUMEL = operator.attrgetter("grad"), torch.Tensor.data_ptr, torch.Tensor.numel           # (for map: a step asks every parameter)
_PARAMS = operator.itemgetter("params")
STEP_ROW = np.dtype([("grad", "<i8"), ("h", "<f4", (8,))])


def _mix(x):
    x ^= x >> 16
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    x ^= x >> 13
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _codes_dtype(second):
    return torch.float8_e5m2 if second else torch.float8_e4m3fn


def _same_layout(a, b):
    return a.stride() == b.stride() and a.shape == b.shape or _same_order(a, b)


def _identical(a, b):
    """The same objects in the same order."""
    return len(a) == len(b) and all(map(operator.is_, a, b))


def _as_now(tensors):
    """An object whose ``check(*tensors)`` says whether size, strides, type and device of every tensor are what they are now: one call for all of
    them (separate questions, one Python call a tensor each, would cost as much as a small step's launches).  Holds no tensor."""
    return TensorGuards(*tensors, dynamic_dims_sizes=[list(t.shape) for t in tensors], dynamic_dims_strides=[list(t.stride()) for t in tensors])


def _memory_order(t):
    """The elements of a dense tensor in memory order (a view)."""
    return t.as_strided((t.numel(),), (1,))


def pack_moment(x, second=False):
    """A moment (fp32, dense) in 8 bits: (codes, scales), codes float8_e4m3fn (first moment) or float8_e5m2 (``second``: >= 0, a positive one
    never becomes 0) of x's shape and memory order, scales uint8, one per 32 elements in memory order: a power of two 2^(scale - 127)
    (255: the block holds a value that is not finite).  value = codes.float() * 2^(scale - 127), rounded to nearest even."""
    if not x.is_cuda:
        raise RuntimeError("moment must be a CUDAtensor ")
    if x.dtype != torch.float32 or not _dense(x):
        raise RuntimeError(f"pack_moment takes a dense float32 tensor (found {x.dtype})")
    x = x.detach()
    codes = torch.empty_like(x, dtype=torch.uint8, memory_format=torch.preserve_format)
    scales = torch.empty(-(-x.numel() // BLOCK), dtype=torch.uint8, device=x.device)
    with _lib.on_device(x.device):
        _lib.call("mmt_moment_pack", x.numel(), x.data_ptr(), int(second), codes.data_ptr(), scales.data_ptr(), _lib.raw_stream(x.device))
    return codes.view(_codes_dtype(second)), scales


def unpack_moment(codes, scales):
    """The fp32 values of (codes, scales) from pack_moment, in the codes' shape and memory order."""
    if not codes.is_cuda or not scales.is_cuda or scales.device != codes.device:
        raise RuntimeError("codes and scales must be CUDAtensors of one device")
    if codes.dtype not in (torch.float8_e4m3fn, torch.float8_e5m2) or scales.dtype != torch.uint8 or not _dense(codes) or not scales.is_contiguous():
        raise RuntimeError(f"unpack_moment takes dense float8_e4m3fn / float8_e5m2 codes and uint8 scales (found {codes.dtype}, {scales.dtype})")
    if scales.numel() != -(-codes.numel() // BLOCK):
        raise RuntimeError(f"unpack_moment: {scales.numel()} scales for {codes.numel()} codes")
    if codes.data_ptr() % 4:
        codes = codes.clone(memory_format=torch.preserve_format)
    out = torch.empty_like(codes, dtype=torch.float32, memory_format=torch.preserve_format)
    with _lib.on_device(codes.device):
        _lib.call("mmt_moment_unpack", codes.numel(), codes.data_ptr(), scales.data_ptr(), int(codes.dtype == torch.float8_e5m2), out.data_ptr(),
                  _lib.raw_stream(codes.device))
    return out


class ClipAdamW8(torch.optim.Optimizer):
    """AdamW with decoupled weight decay and ``clip_grad_norm_`` to ``max_norm`` (the norm over ALL groups; 0: no clipping) over dense fp32 / bf16
    CUDA parameters of one device.

    State of a parameter: ``step``, ``draw`` and, from min_8bit_size elements on, ``exp_avg`` (float8_e4m3fn), ``exp_avg_sq`` (float8_e5m2) in
    the parameter's shape and memory order with ``exp_avg_scale``, ``exp_avg_sq_scale`` (uint8 per 32 elements, see pack_moment); fp32
    moments below.  The moments are views of ``state_buffers()``: to change them, write into them or load a state.  An entry that is
    taken out begins anew.  Parameters join by ``add_param_group`` only.

    The update itself uses unrounded moments; what is stored is rounded stochastically by bits that are a function of ``seed``, the element's
    position and the step's draw: one more than the largest that any parameter taking part has had (``draw``; the step count where all
    have taken part in every step).  So a run repeats exactly, ranks of a data-parallel job agree, and a parameter never meets the bits of
    an earlier step again, whoever joins or leaves.

    A gradient that is infinite or NaN makes NaN of the moments of the 32 elements that share its scale, for good; a NaN under clipping, through
    the norm, of everything.

    ``state_dict()`` resumes exactly (with the same ``seed``).  ``load_state_dict`` also takes the state of torch.optim.AdamW or ClipAdamW
    (32-bit moments are packed), and ``state_dict_32bit()`` hands one to them.  ``last_norm`` holds (total norm, clip coefficient) of
    the last step on the device, a tensor of that step's own; (0, 1) without clipping, which takes no norm.
    ``step()`` cannot be captured into a graph (gradients' addresses and step counts travel from the host): it raises."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=0.0, seed=0, min_8bit_size=4096):
        self._ready, self._plan = False, None
        self._check_hyper(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        if min_8bit_size < 1:
            raise ValueError("ClipAdamW8: min_8bit_size must be at least 1")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.max_norm, self.seed, self.min_8bit_size = float(max_norm), int(seed), int(min_8bit_size)
        self.last_norm = None
        self.shadows = {}       # parameter -> bf16 copy kept current by step() (see make_bf16_shadows)
        self._layout()
        self._ready = True

    @staticmethod
    def _check_hyper(g):
        b1, b2 = g["betas"]
        if not (g["lr"] >= 0.0 and g["eps"] >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and g["weight_decay"] >= 0.0):
            raise ValueError("ClipAdamW8: invalid hyper-parameters")
        if g.get("amsgrad") or g.get("maximize"):
            raise ValueError("ClipAdamW8: amsgrad / maximize are not supported")

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if self._ready:
            try:
                self._layout()
            except Exception:
                self.param_groups.pop()
                raise

    def _packed(self, p):
        return p.numel() >= self.min_8bit_size

    @staticmethod
    def _check_params(ps):
        for p in ps:
            if not (p.is_cuda and p.dtype in (torch.float32, torch.bfloat16) and _dense(p)):
                raise TypeError("ClipAdamW8 takes dense fp32 / bf16 CUDA parameters")
            if p.device != ps[0].device:
                raise TypeError("ClipAdamW8: the parameters are on several devices")

    # ---- the state buffers: one allocation per kind, every parameter's moments a view
    def _layout(self):
        """Gives every parameter its place in new state buffers (again after a group was added: what is there moves along)."""
        ps = [p for g in self.param_groups for p in g["params"]]
        self._check_params(ps)
        for g in self.param_groups:
            self._check_hyper(g)
        held, mine = {p: st for p, st in self.state.items() if "exp_avg" in st}, set(ps)
        for p, st in held.items():
            if p not in mine or "draw" not in st:
                raise RuntimeError("ClipAdamW8: a state is of a parameter that is in no group, or was put there directly (load_state_dict takes states)")
            if not _same_layout(st["exp_avg"], p) or ("exp_avg_scale" in st) != self._packed(p):
                raise RuntimeError("ClipAdamW8: a parameter has changed its size or layout, and its moments (or min_8bit_size) have not")
        n8 = n32 = 0
        place = {}
        for p in ps:
            size = -(-p.numel() // ALIGN) * ALIGN
            if self._packed(p):
                place[p] = (True, n8)
                n8 += size
            else:
                place[p] = (False, n32)
                n32 += size
        self._drop_plan()
        dev = ps[0].device
        u8 = lambda n: torch.zeros(n, dtype=torch.uint8, device=dev)  # noqa: E731
        f32 = lambda n: torch.zeros(n, dtype=torch.float32, device=dev)  # noqa: E731
        buffers = dict(exp_avg=u8(n8), exp_avg_scale=u8(n8 // BLOCK), exp_avg_sq=u8(n8), exp_avg_sq_scale=u8(n8 // BLOCK),
                       exp_avg_32=f32(n32), exp_avg_sq_32=f32(n32))
        self._buffers, self._place, self._params, self._n8 = buffers, place, ps, n8
        self._bases = {key: t.data_ptr() for key, t in buffers.items()}
        self._typed = dict(buffers, exp_avg=buffers["exp_avg"].view(torch.float8_e4m3fn), exp_avg_sq=buffers["exp_avg_sq"].view(torch.float8_e5m2))
        counts, draws = torch.zeros(len(ps), dtype=torch.float32), torch.zeros(len(ps), dtype=torch.int64)
        self._counts, self._draws = counts.numpy(), draws.numpy()             # (the same memory: the states' tensors are views of it)
        self._count_of, self._draw_of = counts.unbind(), draws.unbind()
        self._index = {p: t for t, p in enumerate(ps)}
        self._fill_state(held)
        self._live = [p for p in ps if p.numel()]
        self._empty = [p for p in ps if not p.numel()]
        self._sizes = {p: p.numel() for p in ps}
        self._group_sizes = [len(g["params"]) for g in self.param_groups]
        torch.cuda.current_stream(dev).synchronize()          # (filled on this stream, stepped on whichever)

    def _fill_state(self, states):
        """The parameters' moments and step counts from other tensors of the same form, in the same memory order."""
        to, source = {1: [], 4: []}, {1: [], 4: []}           # by element size: one copy for all the codes and scales, one for all the fp32 moments
        for p, st in states.items():
            self._give_state(p, float(st["step"]), int(st["draw"]))
            packed, at = self._place[p]
            for key in ("exp_avg", "exp_avg_sq"):
                for name, start in ((key, at), (key + "_scale", at // BLOCK)) if packed else ((key, at),):
                    x = st[name]
                    buffer = self._buffers[name if packed else name + "_32"]
                    to[buffer.element_size()].append(buffer.as_strided((x.numel(),), (1,), start))
                    x = x if x.dim() == 1 and x.is_contiguous() else _memory_order(x)
                    source[buffer.element_size()].append(x.view(torch.uint8) if packed and x.dtype != torch.uint8 else x)
        for size in (1, 4):
            if to[size]:
                torch._foreach_copy_(to[size], source[size])

    def _views(self, p):
        packed, at = self._place[p]
        b = self._typed
        if packed:
            blocks = -(-p.numel() // BLOCK)
            return dict(exp_avg=b["exp_avg"].as_strided(p.shape, p.stride(), at), exp_avg_sq=b["exp_avg_sq"].as_strided(p.shape, p.stride(), at),
                        exp_avg_scale=b["exp_avg_scale"].as_strided((blocks,), (1,), at // BLOCK),
                        exp_avg_sq_scale=b["exp_avg_sq_scale"].as_strided((blocks,), (1,), at // BLOCK))
        return dict(exp_avg=b["exp_avg_32"].as_strided(p.shape, p.stride(), at), exp_avg_sq=b["exp_avg_sq_32"].as_strided(p.shape, p.stride(), at))

    def _address(self, p):
        """Where a parameter's first moment begins."""
        packed, at = self._place[p]
        return self._bases["exp_avg"] + at if packed else self._bases["exp_avg_32"] + 4 * at

    def _give_state(self, p, count, draw):
        t = self._index[p]
        self._counts[t], self._draws[t] = count, draw
        self.state[p] = dict(step=self._count_of[t], draw=self._draw_of[t], **self._views(p))

    def state_buffers(self):
        """The buffers that hold all parameters' moments (each parameter's from a multiple of 256 elements on, in the order of the groups, zeros
        between): exp_avg (float8_e4m3fn), exp_avg_sq (float8_e5m2), their scales (uint8), and exp_avg_32 / exp_avg_sq_32 (fp32)."""
        return dict(self._typed)

    @torch.no_grad()
    def make_bf16_shadows(self, params):
        """A bf16 copy of every given fp32 parameter, rewritten by every step() (see ClipAdamW.make_bf16_shadows)."""
        from ..ops import conv_overlap
        for p in params:
            if p.dtype != torch.float32 or p not in self._place:
                raise TypeError("ClipAdamW8: a bf16 copy is kept of this optimizer's fp32 parameters")
            sh = torch.empty_like(p, dtype=torch.bfloat16, memory_format=torch.preserve_format)
            sh.copy_(p)
            self.shadows[p] = sh
            conv_overlap.register_bf16_shadow(p, sh)
        self._drop_plan()

    # ---- tables of the parameters that take part (those with a gradient)
    def _drop_plan(self):
        """(a step queued on another stream may still read the tables and the buffers)"""
        for slot in self._plan["slots"] if self._plan else ():
            if slot["event"] is not None:
                slot["event"].synchronize()
        self._plan = None

    def _tables(self, ps, addresses, grads):
        self._drop_plan()
        dev = self._buffers["exp_avg"].device
        for p, g in zip(ps, grads):                           # (everything but the gradients' addresses is read from the tables until these change)
            if p.device != dev or g.device != dev or p.dtype not in (torch.float32, torch.bfloat16) or not _dense(p):
                raise TypeError(f"ClipAdamW8: a parameter is no longer a dense fp32 / bf16 one on {dev}, or its gradient is elsewhere")
            if p.numel() != self._sizes[p]:
                raise RuntimeError(f"ClipAdamW8: a parameter of {self._sizes[p]} elements has {p.numel()} now (its moments have not)")
            st = self.state[p]
            if "exp_avg" not in st:
                t = self._index[p]
                if self._draws[t]:                            # (it had a state, which the program took out: zeros again, but no bits of the steps before)
                    for x in self._views(p).values():
                        x.view(torch.uint8).zero_() if x.element_size() == 1 else x.zero_()
                self._give_state(p, 0.0, int(self._draws[t]))
            elif st["exp_avg"].data_ptr() != self._address(p):
                raise RuntimeError("ClipAdamW8: a parameter's state was replaced by tensors that are not this optimizer's (load_state_dict takes them)")
            elif not _same_layout(st["exp_avg"], p):
                raise RuntimeError("ClipAdamW8: a moment's layout differs from its parameter's")
            if p in self.shadows and (p.dtype != torch.float32 or not _same_layout(self.shadows[p], p)):
                raise RuntimeError("ClipAdamW8: a parameter's bf16 copy was made for another type or layout of it (make_bf16_shadows makes it anew)")
        total = sum(p.numel() for p in ps)
        chunk = self._chunk(total)
        table = np.zeros((len(ps), COLUMNS), dtype=np.int64)
        base = self._bases
        for t, p in enumerate(ps):
            packed, at = self._place[p]
            if packed:
                row = (base["exp_avg"] + at, base["exp_avg_sq"] + at, base["exp_avg_scale"] + at // BLOCK, base["exp_avg_sq_scale"] + at // BLOCK)
            else:
                row = (base["exp_avg_32"] + 4 * at, base["exp_avg_sq_32"] + 4 * at, 0, 0)
            shadow = self.shadows[p].data_ptr() if p in self.shadows else 0
            table[t] = (addresses[t], *row, shadow, p.numel(), at if packed else self._n8 + at, _lib.DTYPE_BF16 if p.dtype == torch.bfloat16 else _lib.DTYPE_F32)
        each = -(-table[:, 6] // chunk)                       # chunks of every tensor, and each chunk's first element in its tensor
        chunk_t = np.repeat(np.arange(len(ps), dtype=np.int32), each)
        chunk_o = (np.arange(len(chunk_t)) - np.repeat(np.cumsum(each) - each, each)) * chunk
        n_chunks = len(chunk_t)
        partials = _lib.lib().mmt_clip_adamw8_partials(n_chunks)
        slots = []
        for _ in range(RING):   # what a step writes before its kernels have run: the step that takes the slot next waits for its event
            host = torch.empty(len(ps) * STEP_ROW.itemsize, dtype=torch.uint8).pin_memory()
            slots.append(dict(host=host, rows=host.numpy().view(STEP_ROW), device=torch.empty(host.numel(), dtype=torch.uint8, device=dev),
                              partials=torch.empty(partials, dtype=torch.float64, device=dev), event=None))
        group_of = {p: gi for gi, g in enumerate(self.param_groups) for p in g["params"]}
        self._plan = dict(ps=ps, addresses=addresses, n_chunks=n_chunks, chunk=chunk, table=torch.from_numpy(table).to(dev),
                          chunk_t=torch.from_numpy(chunk_t).to(dev), chunk_o=torch.from_numpy(chunk_o).to(dev), slots=slots, turn=0,
                          index=np.array([self._index[p] for p in ps]), group=np.array([group_of[p] for p in ps]),
                          dtypes=[p.dtype for p in ps], states=list(self.state.values()), as_checked=None, streams=set())
        torch.cuda.current_stream(dev).synchronize()          # (built on this stream, read on whichever stream a step runs on)
        return self._plan

    @staticmethod
    def _chunk(total):
        """Elements of a workgroup's turn: 4096 while that makes fewer than 4096 of them (22 us a step of 3.3 M elements; 2048: 23, 1024: 26), else
        8192 (333 us at 84 M; 4096: 338, 16384: 340)."""
        return 4096 if total < 1 << 24 else 8192

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        dev = self._buffers["exp_avg"].device
        if any(map(_NUMEL, self._empty)):
            raise RuntimeError("ClipAdamW8: a parameter that was empty has elements now (its moments have not)")
        with _lib.on_device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("ClipAdamW8.step() cannot be captured into a graph: gradients' addresses and step counts come from the host")
        groups = list(map(_PARAMS, self.param_groups))
        if list(map(len, groups)) != self._group_sizes or not all(map(operator.is_, itertools.chain.from_iterable(groups), self._params)):
            raise RuntimeError("ClipAdamW8: the groups' parameters are not the ones that state was laid out for (add_param_group adds some; for others make a "
                               "new optimizer and load the state)")
        ps = self._live
        grads = list(map(_GRAD, ps))
        try:
            given = list(map(_ADDRESS, grads))
        except (TypeError, RuntimeError):                     # (a parameter without a gradient takes no part; one without storage is refused below)
            ps = [p for p, g in zip(ps, grads) if g is not None]
            grads, given = [g for g in grads if g is not None], None
        if not ps:
            return loss
        addresses = list(map(_ADDRESS, ps))
        plan = self._plan
        if (plan is None or plan["addresses"] != addresses or not (plan["ps"] is ps or _identical(plan["ps"], ps))
                or not _identical(plan["states"], self.state.values())):
            plan = self._tables(ps, addresses, grads)
        # one question for all: is everything as it was when each was last looked at
        if plan["as_checked"] is None or not plan["as_checked"].check(*ps, *grads):
            self._check_each(plan, ps, grads)
            given = None
        with _lib.on_device(dev):
            slot = plan["slots"][plan["turn"]]
            if slot["event"] is not None:
                slot["event"].synchronize()                   # (the step that last used this slot: RING steps ago)
            rows = slot["rows"]
            rows["grad"] = given or list(map(_ADDRESS, grads))
            index = plan["index"]
            counts, draw = self._counts[index] + 1, int(self._draws[index].max()) + 1
            self._fill(rows["h"], plan["group"], counts)
            slot["device"].copy_(slot["host"], non_blocking=True)
            self._counts[index], self._draws[index] = counts, draw
            stream, norm = torch.cuda.current_stream(dev), torch.empty(2, dtype=torch.float32, device=dev)
            _lib.timed_call("clip_adamw8", "mmt_clip_adamw8_step", plan["n_chunks"], plan["chunk"], plan["chunk_t"].data_ptr(), plan["chunk_o"].data_ptr(),
                            plan["table"].data_ptr(), slot["device"].data_ptr(), self._key(draw), self.max_norm,
                            slot["partials"].data_ptr(), norm.data_ptr(), stream.cuda_stream)
            if stream.cuda_stream not in plan["streams"]:
                self._keep_for(stream, plan)
            slot["event"] = slot["event"] or torch.cuda.Event()
            slot["event"].record(stream)
            plan["turn"] = (plan["turn"] + 1) % RING
        self.last_norm = norm
        return loss

    def _keep_for(self, stream, plan):
        """What a step on this stream reads and writes keeps its memory until the stream is done with it, also when the optimizer is dropped before."""
        plan["streams"].add(stream.cuda_stream)
        for t in (*self._buffers.values(), *self.shadows.values(), plan["table"], plan["chunk_t"], plan["chunk_o"],
                  *(slot[key] for slot in plan["slots"] for key in ("device", "partials"))):
            t.record_stream(stream)

    def _check_each(self, plan, ps, grads):
        """Raises unless every parameter is laid out like its moments and has a dense gradient of its shape; gradients of another type or memory order
        are replaced (in ``grads`` and the parameter) by ones of the parameter's."""
        replaced = False
        for i, (p, g) in enumerate(zip(ps, grads)):
            m = self.state[p]["exp_avg"]
            # (a contiguous parameter seen through another shape is still in its moments' order)
            if p.dtype != plan["dtypes"][i] or p.numel() != m.numel() or not (_same_layout(m, p) or m.is_contiguous() and p.is_contiguous()):
                raise RuntimeError("ClipAdamW8: a parameter has changed its size, type or layout in place (its moments have not)")
            if g.shape != p.shape:
                raise RuntimeError(f"ClipAdamW8: a gradient of shape {tuple(g.shape)} for a parameter of shape {tuple(p.shape)}")
            if g.is_sparse:
                raise RuntimeError("ClipAdamW8: a gradient is sparse")
            if g.device != p.device:
                raise TypeError("ClipAdamW8: a gradient is elsewhere than its parameter")
            if g.dtype != p.dtype or not _same_layout(g, p):
                grads[i] = p.grad = torch.empty_like(p).copy_(g)
                replaced = True
        plan["as_checked"] = None if replaced else _as_now(ps + grads)

    def _key(self, draw):
        return _mix((_mix(self.seed & 0xFFFFFFFF) + draw) & 0xFFFFFFFF)

    def _fill(self, h, group, counts):
        """The 8 floats of every tensor: from its group's hyper-parameters and its own step count."""
        def row(g, c):
            (b1, b2), lr = map(float, g["betas"]), float(g["lr"])
            return (1.0 - lr * float(g["weight_decay"]), lr / (1.0 - b1 ** c), b1, 1.0 - b1, b2, 1.0 - b2, 1.0 / math.sqrt(1.0 - b2 ** c), float(g["eps"]))

        if len(self.param_groups) == 1 and (counts == counts[0]).all():
            h[:] = row(self.param_groups[0], float(counts[0]))
            return
        for gi, g in enumerate(self.param_groups):
            mine = group == gi
            for count in np.unique(counts[mine]):
                h[mine & (counts == count)] = row(g, float(count))

    # ---- checkpoints
    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes effect whole or not at all: every moment is checked and converted before anything is replaced."""
        loaded = {}

        def convert(_, sd):                       # last of the pre-hooks: what they made of the state dict is what is loaded
            saved = sd["state"]
            for g in sd["param_groups"]:
                self._check_hyper({**self.defaults, **g})
            order, ps = ([p for g in groups for p in g["params"]] for groups in (sd["param_groups"], self.param_groups))
            if len(order) != len(ps):
                raise ValueError("ClipAdamW8: the state is of another number of parameters")
            self._check_params(ps)
            for k, p in zip(order, ps):
                st = saved.get(k, {})
                if "exp_avg" in st or "exp_avg_sq" in st:
                    loaded[p] = self._loaded(p, st)
            # (a state that does not name its draws was rounded, if at all, by ones up to the largest step count)
            drawn = int(max([0, *(st["step"] for st in loaded.values()), *(st["draw"] for st in loaded.values())]))
            for st in loaded.values():
                st["draw"] = drawn if st["draw"] < 0 else st["draw"]
            return {**sd, "state": {}}

        def install(_):                           # first of the post-hooks: the rest find the moments there
            self._layout()                        # (new buffers: the given tensors may be views of the ones there were)
            self._fill_state(loaded)
            torch.cuda.current_stream(self._buffers["exp_avg"].device).synchronize()

        hooks = self.register_load_state_dict_pre_hook(convert), self.register_load_state_dict_post_hook(install, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _loaded(self, p, st):
        """A parameter's saved state, in the form that it is kept in here."""
        for key in ("step", "exp_avg", "exp_avg_sq"):
            if key not in st:
                raise ValueError(f"ClipAdamW8: a state without {key}")
            if key != "step" and tuple(st[key].shape) != tuple(p.shape):
                raise ValueError(f"ClipAdamW8: {key} of shape {tuple(st[key].shape)} for a parameter of shape {tuple(p.shape)}")
        return dict(step=float(st["step"]), draw=int(st.get("draw", -1)), **self._converted(p, st, "exp_avg"), **self._converted(p, st, "exp_avg_sq"))

    def _converted(self, p, st, key):
        """A saved moment in the form and memory order that this parameter keeps it in: {key: codes, key_scale: scales} or {key: fp32}."""
        x, scales, second = st[key].to(p.device), st.get(key + "_scale"), key == "exp_avg_sq"
        packed = self._packed(p)
        if scales is not None:
            if x.element_size() != 1:
                raise ValueError(f"ClipAdamW8: {key} is {x.dtype} beside its scales, not in 8 bits")
            x, scales = x.view(_codes_dtype(second)), scales.to(p.device)
            if scales.dtype != torch.uint8 or scales.numel() != -(-x.numel() // BLOCK):
                raise ValueError(f"ClipAdamW8: {key}_scale does not fit {key}")
            if packed and _same_layout(x, p):
                return {key: x, key + "_scale": scales}
            x = unpack_moment(x if _dense(x) else x.contiguous(), scales)
        if x.dtype != torch.float32 or not _same_layout(x, p):
            x = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(x)
        return dict(zip((key, key + "_scale"), pack_moment(x, second))) if packed else {key: x}

    @torch.no_grad()
    def state_dict_32bit(self):
        """The state as torch.optim.AdamW and ClipAdamW keep it (fp32 moments): their load_state_dict takes it."""
        sd = self.state_dict()
        state = {}
        for k, st in sd["state"].items():
            state[k] = dict(step=st["step"].clone(), **{
                key: unpack_moment(st[key], st[key + "_scale"]) if key + "_scale" in st else st[key].clone(memory_format=torch.preserve_format)
                for key in ("exp_avg", "exp_avg_sq")})
        return {"state": state, "param_groups": sd["param_groups"]}
