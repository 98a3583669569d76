"""Operators along rays and expert layers on torch tensors (C ABI: the second half of include/ffnerf_hip.h).

They take the packed samples that `ffn_march` leaves.  `RaySet` names them; `ray_attention`, `ray_scan`, `ray_delta`,
`expert_linear`, `expert_dispatch`, `expert_combine` and `layer_norm` compute, their `*_backward` give gradients, and
`RayAttention`, `RayScan`, `RayDelta`, `ExpertLinear`, `ExpertDispatch`, `ExpertCombine`, `LayerNorm` are the same as
functions of torch that can be differentiated once; a second time is an error.  Every call runs on the current stream of its tensors' device, allocates
its results and scratch from torch, and never waits.  A wrong argument is an FfnError before anything is launched.
"""
from __future__ import annotations

import ctypes as C

import torch

import ffn_lib as fl

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _refuse(text: str):
    raise fl.FfnError(text)


def _dtype(x: torch.Tensor) -> int:
    d = DTYPES.get(x.dtype)
    if d is None:
        _refuse(f"dtype {x.dtype} is not float32, float16 or bfloat16")
    return d


def _want(x, name: str, shape: tuple, dtype, dev: int, rows: int = -1) -> int:
    """Pointer of x, which must have this shape, type and device, and (rows -1) be contiguous, (1) have unit stride
    along its last axis, or (0) any strides."""
    if (isinstance(x, torch.Tensor) and x.shape == shape and x.dtype is dtype and x.get_device() == dev
            and (x.is_contiguous() if rows < 0 else not rows or x.stride(-1) == 1 or shape[-1] == 1 or not x.numel())):
        return x.data_ptr()
    if not isinstance(x, torch.Tensor) or x.shape != shape:
        _refuse(f"{name} must be a tensor of shape {tuple(shape)}, not "
                f"{tuple(x.shape) if isinstance(x, torch.Tensor) else type(x).__name__}")
    if x.dtype is not dtype:
        _refuse(f"{name} must be {dtype}, not {x.dtype}")
    if x.get_device() != dev:
        _refuse(f"{name} is on {x.device}, not on cuda:{dev}")
    _refuse(f"{name} must be contiguous" if rows < 0 else f"{name} must have unit stride along its last axis")


def _may(x, *args) -> int | None:
    """_want of a tensor that may be left out."""
    return None if x is None else _want(x, *args)


def _is(x, kind, name: str):
    if not isinstance(x, kind):
        _refuse(f"{name} must be a {kind.__name__}, not {type(x).__name__}")
    return x


def _number(x, name: str) -> float:
    if not isinstance(x, str):
        try:
            return float(x)
        except (TypeError, ValueError):
            pass
    _refuse(f"{name} must be a number, not {type(x).__name__}")


def _index(x, name: str, dev: int) -> int:
    if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.dtype not in (torch.int32, torch.uint32):
        _refuse(f"{name} must be a vector of int32")
    if x.get_device() != dev:
        _refuse(f"{name} is on {x.device}, not on cuda:{dev}")
    if not x.is_contiguous():
        _refuse(f"{name} must be contiguous")
    return x.data_ptr()


class RaySet:
    """Packed rows of rays: ray r has rows offsets[r] .. offsets[r] + counts[r] - 1, ray_ids[i] is row i's ray (all
    int32, as ffn_march leaves them; ray_ids cut to the rows in use).  Rays do not overlap, and all rows of a ray have
    its id; other rows are in no ray."""

    def __init__(self, counts: torch.Tensor, offsets: torch.Tensor, ray_ids: torch.Tensor):
        if not isinstance(ray_ids, torch.Tensor) or not ray_ids.is_cuda:
            _refuse("ray_ids must be a tensor on the GPU")
        dev = self.device = ray_ids.get_device()
        c = self.c = fl.FfnRaySet(_index(counts, "counts", dev), _index(offsets, "offsets", dev),
                                  _index(ray_ids, "ray_ids", dev))
        if counts.shape != offsets.shape:
            _refuse(f"{counts.shape[0]} counts, {offsets.shape[0]} offsets")
        self.num_rays, self.n = counts.shape[0], ray_ids.shape[0]
        if self.num_rays >= 1 << 32 or self.n >= 1 << 31:
            _refuse(f"{self.num_rays} rays with {self.n} rows are too many")
        c.num_rays, c.n = self.num_rays, self.n
        self._keep = (counts, offsets, ray_ids)


def _call(fn, dev: int, *args):
    """fn(*args, stream) on the current stream of device dev."""
    if dev == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        fl.check(rc, fn.__name__)


def _workspace(a, fn, dev: int, *more):
    n = C.c_uint64()
    rc = fn(C.byref(a), *more, C.byref(n))
    if rc:
        fl.check(rc, fn.__name__)
    if not n.value:
        return None
    w = torch.empty(n.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = w.data_ptr(), n.value
    return w


class _Once(torch.autograd.Function):
    """What fn gives, as a function of `inputs` that cannot be differentiated."""

    @staticmethod
    def forward(ctx, fn, *inputs):
        return fn()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the operators' gradients can be differentiated once only: their own gradients are not implemented")


def once(fn, *inputs):
    """fn() of a backward pass that depends on `inputs`.  Under create_graph the results are tied to them, so that a second
    gradient through them is an error, whichever tensors it is asked for; else it would silently lack them."""
    return _Once.apply(fn, *inputs) if torch.is_grad_enabled() else fn()


def _needed(ctx, i: int) -> bool:
    """Whether the gradient of argument i is wanted; one that was left out of the call has none."""
    return i < len(ctx.needs_input_grad) and ctx.needs_input_grad[i]


# ---------------------------------------------------------------------------
# attention


def _attn_args(q, k, v, q_rays, k_rays, t_q, t_k, slopes, scale, cap, causal, prefix):
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or not isinstance(k, torch.Tensor) or k.dim() != 3:
        _refuse("q and k must be tensors [rows, heads, dim]")
    a, dev = fl.FfnRayAttn(), _is(q_rays, RaySet, "q_rays").device
    _is(k_rays, RaySet, "k_rays")
    _, heads, dim = q.shape
    dtype, kv_heads = q.dtype, k.shape[1]
    a.dtype, a.heads, a.kv_heads, a.dim = _dtype(q), heads, kv_heads, dim
    shape = (k_rays.n, kv_heads, dim)
    a.q = _want(q, "q", (q_rays.n, heads, dim), dtype, dev, 1)
    a.k, a.v = _want(k, "k", shape, dtype, dev, 1), _want(v, "v", shape, dtype, dev, 1)
    (a.q_row, a.q_head, _), (a.k_row, a.k_head, _), (a.v_row, a.v_head, _) = q.stride(), k.stride(), v.stride()
    a.q_rays, a.k_rays = q_rays.c, k_rays.c
    a.scale = dim ** -0.5 if scale is None else _number(scale, "scale")
    a.cap, a.causal = _number(cap, "cap"), 1 if causal else 0
    if slopes is not None:
        if t_q is None or t_k is None:
            _refuse("slopes need t_q and t_k")
        a.slopes = _want(slopes, "slopes", (heads,), torch.float32, dev)
        a.t_q = _want(t_q, "t_q", (q_rays.n,), torch.float32, dev, 0)
        a.t_k = _want(t_k, "t_k", (k_rays.n,), torch.float32, dev, 0)
        a.t_q_row, a.t_k_row = t_q.stride(0), t_k.stride(0)
    if prefix is not None:
        a.prefix = _index(prefix, "prefix", dev)
        if prefix.shape[0] != q_rays.num_rays:
            _refuse(f"{prefix.shape[0]} prefixes for {q_rays.num_rays} rays")
        if prefix.dtype == torch.uint32:  # the library's are signed: what is past their end is past any ray's too
            p = prefix.view(torch.int32)
            a.held = torch.where(p < 0, 2 ** 31 - 1, p)  # kept until the launch
            a.prefix = a.held.data_ptr()
    return a, dev


def ray_attention(q, k, v, q_rays: RaySet, k_rays: RaySet | None = None, *, t_q=None, t_k=None, slopes=None,
                  scale: float | None = None, cap: float = 0.0, causal: bool = False, prefix=None):
    """(o, lse): rows of q attend to the rows of k of their own ray.

    q [n_q, heads, dim], k and v [n_k, kv_heads, dim] (float32, float16 or bfloat16, any strides with unit stride along
    dim and 16-byte aligned rows; heads a multiple of kv_heads, which share), dim a multiple of 8 up to 128.  Scores are
    scale q.k (scale: 1/sqrt(dim)), with cap > 0 cap tanh(score / cap), less slopes[head] |t_q - t_k|; causal: a query
    sees no key behind it (places counted from the ray's end where the sets differ), and always the first prefix[ray]
    (int32, below 0 as 0; or uint32).
    k_rays None: q's own set; another one is fast where it holds the rays in the same order.  o as q, lse [n_q, heads]
    float32; a row that sees nothing has 0 and -inf."""
    k_rays = q_rays if k_rays is None else k_rays
    lib = fl.load()
    a, dev = _attn_args(q, k, v, q_rays, k_rays, t_q, t_k, slopes, scale, cap, causal, prefix)
    o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
    a.o, a.lse = o.data_ptr(), lse.data_ptr()
    w = _workspace(a, lib.ffn_ray_attention_workspace, dev, 0)  # noqa: F841 (held until the launch)
    _call(lib.ffn_ray_attention_fwd, dev, C.byref(a))
    return o, lse


def ray_attention_backward(do, q, k, v, o, lse, q_rays: RaySet, k_rays: RaySet | None = None, *, t_q=None, t_k=None,
                           slopes=None, scale: float | None = None, cap: float = 0.0, causal: bool = False, prefix=None):
    """(dq, dk, dv) of ray_attention's o, with its results and the same options."""
    k_rays = q_rays if k_rays is None else k_rays
    lib = fl.load()
    a, dev = _attn_args(q, k, v, q_rays, k_rays, t_q, t_k, slopes, scale, cap, causal, prefix)
    a.o, a.lse = _want(o, "o", q.shape, q.dtype, dev), _want(lse, "lse", q.shape[:2], torch.float32, dev)
    a.dout = _want(do, "do", q.shape, q.dtype, dev, 1)
    a.do_row, a.do_head = do.stride()[:2]
    dq, dk, dv = (torch.empty(x.shape, dtype=q.dtype, device=dev) for x in (q, k, v))
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    w = _workspace(a, lib.ffn_ray_attention_workspace, dev, 1)  # noqa: F841
    _call(lib.ffn_ray_attention_bwd, dev, C.byref(a))
    return dq, dk, dv


class RayAttention(torch.autograd.Function):
    """o of ray_attention; differentiable in q, k and v.  options: a dict of ray_attention's keyword arguments."""

    @staticmethod
    def forward(ctx, q, k, v, q_rays, k_rays=None, options=None):
        ctx.options = options or {}
        ctx.rays = (q_rays, k_rays)
        o, lse = ray_attention(q, k, v, q_rays, k_rays, **ctx.options)
        ctx.save_for_backward(q, k, v, o, lse)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        if do.stride(-1) != 1 or any(s * do.element_size() % 16 for s in do.stride()[:2]) or do.data_ptr() % 16:
            do = do.contiguous()
        grads = once(lambda: ray_attention_backward(do, q, k, v, o, lse, *ctx.rays, **ctx.options), do, q, k, v)
        return (*grads, None, None, None)


# ---------------------------------------------------------------------------
# the gated recurrence


def _scan_args(gate, x, rays, h0, reverse):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        _refuse("x must be a tensor [rows, channels]")
    a, dev = fl.FfnRayScan(), _is(rays, RaySet, "rays").device
    shape = (rays.n, x.shape[1])
    a.dtype, a.channels, a.reverse = _dtype(x), x.shape[1], 1 if reverse else 0
    a.rays = rays.c
    a.gate, a.x = _want(gate, "gate", shape, x.dtype, dev, 1), _want(x, "x", shape, x.dtype, dev, 1)
    a.gate_row, a.x_row = gate.stride(0), x.stride(0)
    a.h0 = _may(h0, "h0", (rays.num_rays, x.shape[1]), torch.float32, dev)
    return a, dev


def ray_scan(gate, x, rays: RaySet, *, h0=None, reverse: bool = False, marks: bool = False):
    """(h, last, marks): h_t = (1 - z_t) h_{t-1} + z_t x_t with z = sigmoid(gate) along each ray, per channel.

    gate and x [n, channels] (float32, float16 or bfloat16, unit stride along the channels); from h0 [num_rays,
    channels] float32 (None: 0); reverse: from each ray's last row to its first, as compositing goes.  h as x; last
    [num_rays, channels] float32, the state after each ray; marks: what ray_scan_backward needs (None unless asked)."""
    lib = fl.load()
    a, dev = _scan_args(gate, x, rays, h0, reverse)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    last = torch.empty((rays.num_rays, x.shape[1]), dtype=torch.float32, device=dev)
    a.h, a.last = h.data_ptr(), last.data_ptr()
    m = None
    if marks:
        n = C.c_uint64()
        fl.check(lib.ffn_ray_scan_marks(C.byref(a), C.byref(n)), "ffn_ray_scan_marks")
        m = torch.empty(n.value // 4, dtype=torch.float32, device=dev)
        a.marks = m.data_ptr()
    w = _workspace(a, lib.ffn_ray_scan_workspace, dev, 0)  # noqa: F841
    _call(lib.ffn_ray_scan_fwd, dev, C.byref(a))
    return h, last, m


def ray_scan_backward(dh, gate, x, marks, rays: RaySet, *, dlast=None, h0=None, reverse: bool = False):
    """(dgate, dx, dh0) of ray_scan's h (dh) and last (dlast, None: 0), with its marks."""
    lib = fl.load()
    a, dev = _scan_args(gate, x, rays, h0, reverse)
    a.dh = _want(dh, "dh", x.shape, x.dtype, dev, 1)
    a.dh_row = dh.stride(0)
    a.dlast = _may(dlast, "dlast", (rays.num_rays, x.shape[1]), torch.float32, dev)
    n = C.c_uint64()
    fl.check(lib.ffn_ray_scan_marks(C.byref(a), C.byref(n)), "ffn_ray_scan_marks")
    a.marks = _may(marks, "marks", (n.value // 4,), torch.float32, dev)
    dgate, dx = torch.empty(x.shape, dtype=x.dtype, device=dev), torch.empty(x.shape, dtype=x.dtype, device=dev)
    dh0 = torch.empty((rays.num_rays, x.shape[1]), dtype=torch.float32, device=dev)
    a.dgate, a.dx, a.dh0 = dgate.data_ptr(), dx.data_ptr(), dh0.data_ptr()
    w = _workspace(a, lib.ffn_ray_scan_workspace, dev, 1)  # noqa: F841
    _call(lib.ffn_ray_scan_bwd, dev, C.byref(a))
    return dgate, dx, dh0


class RayScan(torch.autograd.Function):
    """(h, last) of ray_scan; differentiable in gate, x and h0."""

    @staticmethod
    def forward(ctx, gate, x, rays, h0=None, reverse=False):
        h, last, marks = ray_scan(gate, x, rays, h0=h0, reverse=reverse, marks=True)
        ctx.save_for_backward(gate, x, marks, h0)
        ctx.rays, ctx.reverse = rays, reverse
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        gate, x, marks, h0 = ctx.saved_tensors
        dh = dh if dh.stride(-1) == 1 else dh.contiguous()
        dgate, dx, dh0 = once(lambda: ray_scan_backward(dh, gate, x, marks, ctx.rays, dlast=dlast.contiguous(), h0=h0,
                                                        reverse=ctx.reverse), dh, dlast, gate, x, h0)
        return dgate, dx, None, (dh0 if h0 is not None else None), None


# ---------------------------------------------------------------------------
# the delta rule


def _delta_args(q, k, v, decay, beta, rays, h0, scale, reverse):
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or not isinstance(v, torch.Tensor) or v.dim() != 3:
        _refuse("q and v must be tensors [rows, heads, dim]")
    a, dev = fl.FfnRayDelta(), _is(rays, RaySet, "rays").device
    n, dtype = rays.n, q.dtype
    (_, heads, dk), (_, v_heads, dv) = q.shape, v.shape
    a.dtype, a.heads, a.v_heads, a.key_dim, a.val_dim = _dtype(q), heads, v_heads, dk, dv
    a.reverse, a.rays = 1 if reverse else 0, rays.c
    a.scale = dk ** -0.5 if scale is None and dk else _number(scale, "scale")
    a.q, a.k = _want(q, "q", (n, heads, dk), dtype, dev, 1), _want(k, "k", (n, heads, dk), dtype, dev, 1)
    a.v = _want(v, "v", (n, v_heads, dv), dtype, dev, 1)
    a.decay = _want(decay, "decay", (n, v_heads), dtype, dev, 0)
    a.beta = _want(beta, "beta", (n, v_heads), dtype, dev, 0)
    (a.q_row, a.q_head, _), (a.k_row, a.k_head, _), (a.v_row, a.v_head, _) = q.stride(), k.stride(), v.stride()
    (a.decay_row, a.decay_head), (a.beta_row, a.beta_head) = decay.stride(), beta.stride()
    state = (rays.num_rays, v_heads, dk, dv)
    a.h0 = _may(h0, "h0", state, torch.float32, dev)
    return a, dev, state


def ray_delta(q, k, v, decay, beta, rays: RaySet, *, h0=None, scale: float | None = None, reverse: bool = False,
              last=False, marks: bool = False):
    """(o, last, marks): a matrix state a ray and value head, S_t = a_t S_{t-1} + k_t n_t^T with a_t = exp(decay_t) and
    n_t = beta_t (v_t - a_t S_{t-1}^T k_t), read as o_t = scale S_t^T q_t (scale: 1/sqrt(key dim)).

    q and k [n, heads, key_dim], v [n, v_heads, val_dim] (float32, float16 or bfloat16, unit stride along the dims, rows
    and heads on 16 bytes, rows less than 16 MiB apart; v_heads a multiple of heads, which are shared; dims multiples of 8
    up to 128), decay (at most 0; -inf forgets what was before) and beta [n, v_heads] of the same type; stable where
    beta |k|^2 <= 2.  From h0 [num_rays, v_heads, key_dim, val_dim] float32 (None: 0); reverse: from each ray's last row to
    its first.  o [n, v_heads, val_dim];
    last: True for the state after each ray, or a tensor that takes it (h0 itself: in place), as h0; marks: what
    ray_delta_backward needs (refused with h0 in place, which the backward reads too).  Both None unless asked."""
    lib = fl.load()
    a, dev, state = _delta_args(q, k, v, decay, beta, rays, h0, scale, reverse)
    o = torch.empty(v.shape, dtype=v.dtype, device=dev)
    given = isinstance(last, torch.Tensor)
    if given:
        a.last = _want(last, "last", state, torch.float32, dev)
    else:
        last = torch.empty(state, dtype=torch.float32, device=dev) if last else None
        a.last = last.data_ptr() if last is not None else None
    a.o, m = o.data_ptr(), None
    if marks:
        n = C.c_uint64()
        fl.check(lib.ffn_ray_delta_marks(C.byref(a), C.byref(n)), "ffn_ray_delta_marks")
        m = torch.empty(n.value // 4, dtype=torch.float32, device=dev)
        a.marks = m.data_ptr()
    _call(lib.ffn_ray_delta_fwd, dev, C.byref(a))
    if given and not last.is_inference():
        torch.autograd.graph.increment_version(last)  # a backward pass that has saved it must not use what is there now
    return o, last, m


def ray_delta_backward(do, q, k, v, decay, beta, marks, rays: RaySet, *, dlast=None, h0=None, scale: float | None = None,
                       reverse: bool = False):
    """(dq, dk, dv, ddecay, dbeta, dh0) of ray_delta's o (do) and last (dlast, None: 0), with its marks and options.  Of the
    inputs' type; dh0 float32, None without h0.  ddecay is a sum of products and exact to their size: relative to itself that
    is less where a decay is strong (some 1e-3 at -8, nothing from -16 on); it is 0 at -inf."""
    lib = fl.load()
    a, dev, state = _delta_args(q, k, v, decay, beta, rays, h0, scale, reverse)
    a.dout = _want(do, "do", v.shape, v.dtype, dev, 1)
    a.do_row, a.do_head = do.stride()[:2]
    a.dlast = _may(dlast, "dlast", state, torch.float32, dev)
    n = C.c_uint64()
    fl.check(lib.ffn_ray_delta_marks(C.byref(a), C.byref(n)), "ffn_ray_delta_marks")
    a.marks = _want(marks, "marks", (n.value // 4,), torch.float32, dev)
    out = [torch.empty(x.shape, dtype=q.dtype, device=dev) for x in (q, k, v, decay, beta)]
    a.dq, a.dk, a.dv, a.ddecay, a.dbeta = (x.data_ptr() for x in out)
    dh0 = torch.empty(state, dtype=torch.float32, device=dev) if h0 is not None else None
    a.dh0 = dh0.data_ptr() if h0 is not None else None
    w = _workspace(a, lib.ffn_ray_delta_workspace, dev, 1)  # noqa: F841
    _call(lib.ffn_ray_delta_bwd, dev, C.byref(a))
    return (*out, dh0)


class RayDelta(torch.autograd.Function):
    """(o, last) of ray_delta; differentiable in q, k, v, decay, beta and h0.  options: a dict of scale and reverse, and
    last=False where the state after the rays is not wanted (None).  Marks are made where a gradient is wanted only."""

    @classmethod
    def apply(cls, q, k, v, decay, beta, rays, h0=None, options=None):
        return super().apply(q, k, v, decay, beta, rays, h0, options, torch.is_grad_enabled())

    @staticmethod
    def forward(ctx, q, k, v, decay, beta, rays, h0, options, grads):
        ctx.options = dict(options or {})
        wanted = ctx.options.pop("last", True)
        o, last, marks = ray_delta(q, k, v, decay, beta, rays, h0=h0, last=bool(wanted),
                                   marks=grads and any(ctx.needs_input_grad), **ctx.options)
        ctx.save_for_backward(q, k, v, decay, beta, marks, h0)
        ctx.rays = rays
        return o, last

    @staticmethod
    def backward(ctx, do, dlast):
        q, k, v, decay, beta, marks, h0 = ctx.saved_tensors
        b = do.element_size()
        if (do.stride(-1) != 1 or any(s * b % 16 for s in do.stride()[:2]) or do.data_ptr() % 16
                or do.stride(0) * b >= fl.DELTA_ROW_BYTES):
            do = do.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        dq, dk, dv, dg, db, dh0 = once(
            lambda: ray_delta_backward(do, q, k, v, decay, beta, marks, ctx.rays, dlast=dlast, h0=h0, **ctx.options),
            do, dlast, q, k, v, decay, beta, h0)
        return dq, dk, dv, dg, db, None, dh0, None, None


# ---------------------------------------------------------------------------
# expert layers


class ExpertPlan:
    """Rows grouped by expert.  counts and offsets [n_experts] and rows [n] (int32): group e is rows[offsets[e] :
    offsets[e] + counts[e]], in the rows' own order; rows of no expert come last."""

    def __init__(self, words: torch.Tensor, n: int, n_experts: int):
        self.words, self.n, self.n_experts, self.device = words, n, n_experts, words.get_device()

    @property
    def counts(self) -> torch.Tensor:
        return self.words[:self.n_experts]

    @property
    def offsets(self) -> torch.Tensor:
        return self.words[self.n_experts + 1:2 * self.n_experts + 1]

    @property
    def rows(self) -> torch.Tensor:
        return self.words[self.words.shape[0] - self.n:]


def _plan(ids, n_experts, slots):
    """The plan of ids, a flat tensor of int32 on the GPU, and (given) the slot of each place."""
    lib = fl.load()
    if not hasattr(n_experts, "__index__") or not 1 <= n_experts <= fl.MAX_EXPERTS:
        _refuse(f"n_experts={n_experts!r} must be a whole number of 1 to {fl.MAX_EXPERTS}")
    dev, n = ids.get_device(), ids.numel()
    if n >= 1 << 31:
        _refuse(f"{n} rows are too many")
    words, ws = C.c_uint64(), C.c_uint64()
    fl.check(lib.ffn_expert_plan_size(n, n_experts, C.byref(words), C.byref(ws)), "ffn_expert_plan_size")
    plan = torch.empty(words.value, dtype=torch.int32, device=dev)
    w = torch.empty(ws.value, dtype=torch.uint8, device=dev) if ws.value else None
    scratch = (None if w is None else w.data_ptr(), ws.value)
    if slots is None:
        _call(lib.ffn_expert_plan, dev, ids.data_ptr(), n, n_experts, plan.data_ptr(), words.value, *scratch)
    else:
        _call(lib.ffn_expert_route, dev, ids.data_ptr(), n, n_experts, plan.data_ptr(), words.value, slots.data_ptr(), *scratch)
    return ExpertPlan(plan, n, n_experts)


def expert_plan(ids: torch.Tensor, n_experts: int) -> ExpertPlan:
    """Groups rows by the expert ids [n] (int32) of the rows; an id outside [0, n_experts) gives a row to none."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dim() != 1 or ids.dtype != torch.int32:
        _refuse("ids must be a vector of int32 on the GPU")
    _index(ids, "ids", ids.get_device())
    return _plan(ids, n_experts, None)


def _expert_args(x, W, plan, relu, x_slots, y_slots):
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not isinstance(W, torch.Tensor) or W.dim() != 3:
        _refuse("x must be a tensor [rows, in], W a tensor [experts, out, in]")
    a, dev = fl.FfnExperts(), _is(plan, ExpertPlan, "plan").device
    a.dtype, a.n_experts, a.d_in, a.d_out = _dtype(x), plan.n_experts, W.shape[2], W.shape[1]
    a.relu, a.flags = 1 if relu else 0, (1 if x_slots else 0) | (2 if y_slots else 0)
    a.n, a.plan = plan.n, plan.words.data_ptr()
    a.x, a.x_row = _want(x, "x", (plan.n, W.shape[2]), x.dtype, dev, 1), x.stride(0)
    a.W = _want(W, "W", (plan.n_experts, W.shape[1], W.shape[2]), x.dtype, dev)
    return a, dev


def expert_linear(x, W, b, plan: ExpertPlan, *, relu: bool = False, x_slots: bool = False, y_slots: bool = False):
    """y = act(x W_e^T + b_e) with each row's expert e.

    x [n, in] (float32, float16 or bfloat16; unit stride along in, 16-byte aligned rows), W [experts, out, in], b
    [experts, out] or None; in and out multiples of 8 up to 4096.  x_slots, y_slots: x, or y, is in the plan's slot
    order instead of the rows' own.  y [n, out]; rows of no expert give 0."""
    lib = fl.load()
    a, dev = _expert_args(x, W, plan, relu, x_slots, y_slots)
    a.b = _may(b, "b", W.shape[:2], x.dtype, dev)
    y = torch.empty((plan.n, W.shape[1]), dtype=x.dtype, device=dev)
    a.y = y.data_ptr()
    _call(lib.ffn_expert_linear_fwd, dev, C.byref(a))
    return y


def expert_linear_backward(dy, x, W, plan: ExpertPlan, *, y=None, x_slots: bool = False, y_slots: bool = False,
                           need_dx: bool = True, need_dw: bool = True):
    """(dx, dW, db) of expert_linear; y: the forward's output of a relu layer (None: no relu).  dx as x, dW and db
    float32; None for those not needed."""
    lib = fl.load()
    a, dev = _expert_args(x, W, plan, y is not None, x_slots, y_slots)
    shape = (plan.n, W.shape[1])
    a.y, a.dy, a.dy_row = _may(y, "y", shape, x.dtype, dev), _want(dy, "dy", shape, x.dtype, dev, 1), dy.stride(0)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_dx else None
    dW = torch.empty(W.shape, dtype=torch.float32, device=dev) if need_dw else None
    db = torch.empty(W.shape[:2], dtype=torch.float32, device=dev) if need_dw else None
    a.dx, a.dW, a.db = (t.data_ptr() if t is not None else None for t in (dx, dW, db))
    w = _workspace(a, lib.ffn_expert_linear_workspace, dev)  # noqa: F841
    _call(lib.ffn_expert_linear_bwd, dev, C.byref(a))
    return dx, dW, db


class ExpertLinear(torch.autograd.Function):
    """expert_linear; differentiable in x, W and b."""

    @staticmethod
    def forward(ctx, x, W, b, plan, relu=False, x_slots=False, y_slots=False):
        y = expert_linear(x, W, b, plan, relu=relu, x_slots=x_slots, y_slots=y_slots)
        ctx.save_for_backward(x, W, y if relu else None)
        ctx.plan, ctx.order, ctx.bias = plan, dict(x_slots=x_slots, y_slots=y_slots), b is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, W, y = ctx.saved_tensors
        if dy.stride(-1) != 1 or dy.stride(0) * dy.element_size() % 16 or dy.data_ptr() % 16:
            dy = dy.contiguous()
        need_dw = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dW, db = once(lambda: expert_linear_backward(dy, x, W, ctx.plan, y=y, need_dx=ctx.needs_input_grad[0],
                                                         need_dw=need_dw, **ctx.order), dy, x, W)
        return (dx, dW.to(W.dtype) if need_dw else None, db.to(W.dtype) if need_dw and ctx.bias else None, None, None,
                None, None)


# ---------------------------------------------------------------------------
# rows to several experts and back


class ExpertRoute:
    """Rows that go to k experts each.  plan: the ExpertPlan of the n k places, place i k + j being row i's j-th expert;
    slots [n, k] (int32): the plan's slot of each place.  Arrays "of slots" have n k rows in the plan's order, as
    expert_linear takes and gives them with x_slots and y_slots; slots of no expert come last."""

    def __init__(self, plan: ExpertPlan, slots: torch.Tensor):
        self.plan, self.slots, self.device = plan, slots, plan.device
        self.n, self.k = slots.shape


def expert_route(ids: torch.Tensor, n_experts: int) -> ExpertRoute:
    """The route of rows with expert ids [n, k] (int32); an id outside [0, n_experts) leaves its place without an expert."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dim() != 2 or ids.dtype != torch.int32:
        _refuse("ids must be a matrix [rows, k] of int32 on the GPU")
    if not ids.is_contiguous():
        _refuse("ids must be contiguous")
    if not 1 <= ids.shape[1] <= fl.MAX_EXPERTS:
        _refuse(f"k={ids.shape[1]} must be 1 to {fl.MAX_EXPERTS}")
    slots = torch.empty(ids.shape, dtype=torch.int32, device=ids.device)
    return ExpertRoute(_plan(ids, n_experts, slots), slots)


def _route_args(x, name, route, slots: bool, weights=None):
    """Arguments with the width and type of x, an array of rows or of slots."""
    dev = _is(route, ExpertRoute, "route").device
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        _refuse(f"{name} must be a tensor [{'slots' if slots else 'rows'}, width]")
    a = fl.FfnRoute()
    a.dtype, a.n_experts, a.k, a.width, a.n = _dtype(x), route.plan.n_experts, route.k, x.shape[1], route.n
    a.plan, a.slots = route.plan.words.data_ptr(), route.slots.data_ptr()
    at = _want(x, name, (route.n * route.k if slots else route.n, x.shape[1]), x.dtype, dev, 1)
    if slots:
        a.slots_in, a.slots_stride = at, x.stride(0)
    else:
        a.rows_in, a.rows_stride = at, x.stride(0)
    a.weights = _may(weights, "weights", (route.n, route.k), torch.float32, dev)
    return a, dev


def expert_dispatch(x, route: ExpertRoute):
    """Rows of x [n, width] (float32, float16 or bfloat16, unit stride along the columns) in the slots' order [n k, width];
    slots of no expert are 0."""
    a, dev = _route_args(x, "x", route, False)
    out = torch.empty((route.n * route.k, x.shape[1]), dtype=x.dtype, device=dev)
    a.slots_out = out.data_ptr()
    _call(fl.load().ffn_expert_dispatch, dev, C.byref(a))
    return out


def expert_dispatch_backward(dxs, route: ExpertRoute):
    """dx [n, width] of expert_dispatch from the gradient of its slots: each row's slots, summed."""
    return expert_combine(dxs, route)


def expert_combine(y, route: ExpertRoute, weights=None):
    """Sums back to rows [n, width]: sum_j weights[i, j] y[slot of row i's j-th expert].

    y [n k, width] of slots (float32, float16 or bfloat16, unit stride along the columns), weights [n, k] float32 (None:
    1).  Sums are float32; a place of no expert adds nothing, whatever y and weights hold there."""
    a, dev = _route_args(y, "y", route, True, weights)
    out = torch.empty((route.n, y.shape[1]), dtype=y.dtype, device=dev)
    a.rows_out = out.data_ptr()
    _call(fl.load().ffn_expert_combine, dev, C.byref(a))
    return out


def expert_combine_backward(dout, y, route: ExpertRoute, weights=None, *, need_dweights: bool = True):
    """(dy, dweights) of expert_combine: dy of slots (0 in those of no expert), dweights [n, k] float32 (0 at places of no
    expert; None if not needed)."""
    a, dev = _route_args(dout, "dout", route, False, weights)
    if need_dweights:
        a.slots_in = _want(y, "y", (route.n * route.k, dout.shape[1]), dout.dtype, dev, 1)
        a.slots_stride = y.stride(0)
    dy = torch.empty((route.n * route.k, dout.shape[1]), dtype=dout.dtype, device=dev)
    dw = torch.empty((route.n, route.k), dtype=torch.float32, device=dev) if need_dweights else None
    a.slots_out, a.dweights = dy.data_ptr(), (dw.data_ptr() if need_dweights else None)
    _call(fl.load().ffn_expert_combine_bwd, dev, C.byref(a))
    return dy, dw


class ExpertDispatch(torch.autograd.Function):
    """expert_dispatch; differentiable in x."""

    @staticmethod
    def forward(ctx, x, route):
        ctx.route = route
        return expert_dispatch(x, route)

    @staticmethod
    def backward(ctx, dxs):
        dxs = dxs if dxs.stride(-1) == 1 else dxs.contiguous()
        return once(lambda: expert_dispatch_backward(dxs, ctx.route), dxs), None


class ExpertCombine(torch.autograd.Function):
    """expert_combine; differentiable in y and weights."""

    @staticmethod
    def forward(ctx, y, route, weights=None):
        ctx.route = route
        ctx.save_for_backward(y, weights)
        return expert_combine(y, route, weights)

    @staticmethod
    def backward(ctx, dout):
        y, weights = ctx.saved_tensors
        dout = dout if dout.stride(-1) == 1 else dout.contiguous()
        need = _needed(ctx, 2)
        dy, dw = once(lambda: expert_combine_backward(dout, y, ctx.route, weights, need_dweights=need), dout, y, weights)
        return dy, None, dw


# ---------------------------------------------------------------------------
# layer norm


def _norm_args(x, weight, bias, eps):
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 2:
        _refuse("x must be a tensor [rows, width] on the GPU")
    a, dev = fl.FfnNorm(), x.get_device()
    if x.shape[0] >= 1 << 31:
        _refuse(f"{x.shape[0]} rows are too many")
    given = [p for p in (weight, bias) if isinstance(p, torch.Tensor)]
    kind = torch.float32 if any(p.dtype is torch.float32 for p in given) else x.dtype
    a.dtype, a.param_dtype, a.width, a.n, a.eps = _dtype(x), DTYPES[kind], x.shape[1], x.shape[0], _number(eps, "eps")
    a.x, a.x_row = _want(x, "x", tuple(x.shape), x.dtype, dev, 1), x.stride(0)
    a.weight = _may(weight, "weight", (x.shape[1],), kind, dev)
    a.bias = _may(bias, "bias", (x.shape[1],), kind, dev)
    return a, dev


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias by rows, rstd = 1 / sqrt(var + eps).

    x [n, width] (float32, float16 or bfloat16, unit stride along the columns; fastest where rows start on 16 bytes), width
    up to 16384; weight and bias [width] both float32 or both of x's type (None: 1 and 0).  y as x; mean and rstd [n]
    float32."""
    a, dev = _norm_args(x, weight, bias, eps)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean, rstd = (torch.empty(x.shape[0], dtype=torch.float32, device=dev) for _ in range(2))
    a.y, a.mean, a.rstd = y.data_ptr(), mean.data_ptr(), rstd.data_ptr()
    _call(fl.load().ffn_layer_norm_fwd, dev, C.byref(a))
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, *, need_dx: bool = True, need_dw: bool = True):
    """(dx, dweight, dbias) of layer_norm, with its mean and rstd.  dx as x, dweight and dbias [width] float32; None for
    those not needed."""
    a, dev = _norm_args(x, weight, None, 0.0)
    a.dy, a.dy_row = _want(dy, "dy", tuple(x.shape), x.dtype, dev, 1), dy.stride(0)
    a.mean = _want(mean, "mean", (x.shape[0],), torch.float32, dev)
    a.rstd = _want(rstd, "rstd", (x.shape[0],), torch.float32, dev)
    lib = fl.load()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_dx else None
    dw, db = (torch.empty(x.shape[1], dtype=torch.float32, device=dev) if need_dw else None for _ in range(2))
    a.dx, a.dweight, a.dbias = (t.data_ptr() if t is not None else None for t in (dx, dw, db))
    w = _workspace(a, lib.ffn_layer_norm_workspace, dev) if need_dw else None  # noqa: F841
    _call(lib.ffn_layer_norm_bwd, dev, C.byref(a))
    return dx, dw, db


class LayerNorm(torch.autograd.Function):
    """y of layer_norm; differentiable in x, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        y, mean, rstd = layer_norm(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dy = dy if dy.stride(-1) == 1 else dy.contiguous()
        need_w, need_b = _needed(ctx, 1), _needed(ctx, 2)
        dx, dw, db = once(lambda: layer_norm_backward(dy, x, weight, mean, rstd, need_dx=ctx.needs_input_grad[0],
                                                      need_dw=need_w or need_b), dy, x, weight)
        return dx, dw.to(weight.dtype) if need_w else None, db.to(ctx.bias_dtype) if need_b else None, None
