"""Device-memory entry points over torch tensors (PyTorch = allocator + streams).

Each function builds the unpacked memref descriptors the C ABI expects from a
CUDA tensor (aligned pointer = tensor.data_ptr(), offset 0, sizes and strides
in elements) and calls the matching spmdb200_* entry on the current stream.
All compute happens in libspmdb200.so; nothing here computes anything.
"""
from __future__ import annotations

import ctypes
import math
from array import array

import torch

from ._lib import c_i, c_p, call, lib
from .forall_program import insn as map_insn  # noqa: F401  (re-exported)

_DTYPES = {torch.float32: "f32", torch.int32: "i32", torch.uint8: "u8", torch.float64: "f64"}


def memref(t: torch.Tensor) -> tuple:
    """Unpacked memref descriptor (base, aligned, offset, sizes..., strides...)."""
    if not t.is_cuda:
        raise ValueError("device entries take CUDA tensors")
    if t.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {t.dtype}")
    p = c_p(t.data_ptr())
    return (p, p, c_i(0), *[c_i(s) for s in t.shape], *[c_i(s) for s in t.stride()])


def _stream(stream) -> c_p:
    s = torch.cuda.current_stream() if stream is None else stream
    return c_p(s.cuda_stream)


def ewise(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """out = a + b (f32), the ewise_kernel forall."""
    n = a.shape[0]
    out = torch.empty_like(a) if out is None else out
    call("spmdb200_ewise", *memref(a), *memref(b), *memref(out), c_i(n), _stream(stream))
    return out


def axpy(alpha: float, x: torch.Tensor, y: torch.Tensor, stream=None) -> torch.Tensor:
    """y = fadd(fmul(alpha, x), y) in place."""
    call("spmdb200_axpy", ctypes.c_float(alpha), *memref(x), *memref(y), c_i(x.shape[0]), _stream(stream))
    return y


def stencil3pt(a: torch.Tensor, out: torch.Tensor, n: int | None = None, m: int | None = None,
               stream=None) -> torch.Tensor:
    """out[i,j] = (a[i,j] + a[i,j+1]) + a[i+1,j] for i < n, j < m (reads off `a` are 0)."""
    n = out.shape[0] if n is None else n
    m = out.shape[1] if m is None else m
    call("spmdb200_stencil3pt", *memref(a), *memref(out), c_i(n), c_i(m), _stream(stream))
    return out


PLAN_REASONS = {0: "promote", 1: "unbounded offsets", 2: "read-write operand", 3: "footprint too large",
                4: "no reuse"}


def _i64(vals) -> ctypes.Array:
    vals = [int(v) for v in vals]
    return (ctypes.c_int64 * max(len(vals), 1))(*vals)


def promotion_plan(tile_sizes, min_offsets, max_offsets, steps=None, elem_bytes: int = 4,
                   max_group_bytes: int = 49152, read_only: bool = True) -> tuple[int, tuple, int]:
    """(plan code, footprint extents, footprint bytes) of one operand, as the
    reference's computePromotionPlan decides it (host only, no GPU needed)."""
    rank = len(tile_sizes)
    dims = (ctypes.c_int64 * 3)()
    nbytes = ctypes.c_int64(0)
    code = lib().spmdb200_promotion_plan(rank, _i64(tile_sizes), _i64(steps) if steps is not None else None,
                                         _i64(min_offsets), _i64(max_offsets), c_i(elem_bytes),
                                         c_i(max_group_bytes), int(bool(read_only)), dims, ctypes.byref(nbytes))
    if code < 0:
        from ._lib import check
        check("spmdb200_promotion_plan", code)  # raises with the library's message
    return int(code), tuple(int(dims[d]) for d in range(rank)), int(nbytes.value)


def stencil_nd(a: torch.Tensor, out: torch.Tensor, offsets, weights=None, scale: float = 1.0, tile_sizes=None,
               steps=None, max_group_bytes: int = 0, policy: int = 0, stream=None) -> bool:
    """out[p] = scale * sum_k w_k * a[p + offsets[k]] in order, for p on the step
    lattice inside out's shape (reads off `a` are 0).  Returns True when the
    promotion plan staged tiles in shared memory."""
    rank = a.dim()
    if out.dim() != rank or not (1 <= rank <= 3):
        raise ValueError("a and out must have the same rank, 1-3")
    offs = [int(v) for row in offsets for v in (row if hasattr(row, "__len__") else [row])]
    ntaps = len(offs) // rank
    tile_sizes = tile_sizes or ([256] if rank == 1 else [32, 8] if rank == 2 else [8, 8, 4])
    w = None if weights is None else (ctypes.c_float * ntaps)(*[float(x) for x in weights])
    promoted = ctypes.c_int(0)
    call("spmdb200_stencil_nd", rank, c_p(a.data_ptr()), _i64(a.shape), _i64(a.stride()), c_p(out.data_ptr()),
         _i64(out.shape), _i64(out.stride()), ntaps, _i64(offs), w, ctypes.c_float(scale), _i64(tile_sizes),
         _i64(steps) if steps is not None else None, c_i(max_group_bytes), policy, ctypes.byref(promoted),
         _stream(stream))
    return bool(promoted.value)


def forall_map(inputs, out: torch.Tensor, code, consts=(), n_regs: int | None = None, stream=None) -> torch.Tensor:
    """out[p] = f(inputs[0][p], ...) over out's domain (rank 1-3), f the
    straight-line program `code` (a list of forall_program.insn pairs; LOADs
    first, one STORE last).  Each input is a view with out's shape."""
    rank = out.dim()
    if not 1 <= rank <= 3:
        raise ValueError("forall_map: rank 1-3")
    for t in inputs:
        if tuple(t.shape) != tuple(out.shape) or t.dtype != torch.float32 or not t.is_cuda:
            raise ValueError("forall_map: every input is a CUDA f32 view with out's shape")
    if out.dtype != torch.float32 or not out.is_cuda:
        raise ValueError("forall_map: out must be a CUDA f32 tensor")
    words = [int(w) for ins in code for w in ins]
    if n_regs is None:
        n_regs = 1 + max(max((w0 >> 8) & 255, (w0 >> 16) & 255, (w0 >> 24) & 255) for w0 in words[0::2])
    ptrs = (c_p * max(len(inputs), 1))(*[t.data_ptr() for t in inputs])
    strides = _i64([s for t in inputs for s in t.stride()] or [0])
    cs = (ctypes.c_float * max(len(consts), 1))(*[float(c) for c in consts])
    call("spmdb200_forall_map", rank, _i64(out.shape), len(inputs), ptrs, strides, c_p(out.data_ptr()),
         _i64(out.stride()), (ctypes.c_int32 * len(words))(*words), len(code), cs, len(consts), n_regs,
         _stream(stream))
    return out


def sum_workspace(n: int, device=None) -> torch.Tensor:
    """Zero-filled workspace for sum_f32 (reusable: every call leaves it zeroed)."""
    nbytes = int(lib().spmdb200_sum_workspace_bytes(c_i(n)))
    return torch.zeros(nbytes, dtype=torch.uint8, device=device or "cuda")


def sum_f32(a: torch.Tensor, out: torch.Tensor, ws: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """out[0] = f32(f64(out[0]) + sum(a)), deterministic."""
    n = a.shape[0]
    ws = sum_workspace(n, a.device) if ws is None else ws
    o = c_p(out.data_ptr())
    call("spmdb200_sum_f32", *memref(a), o, o, c_i(0), c_i(n), c_p(ws.data_ptr()), ctypes.c_size_t(ws.numel()),
         _stream(stream))
    return out


def sum_i32(a: torch.Tensor, out: torch.Tensor, stream=None) -> torch.Tensor:
    """out[0] += sum(a) in wrapping int32."""
    o = c_p(out.data_ptr())
    call("spmdb200_sum_i32", *memref(a), o, o, c_i(0), c_i(a.shape[0]), _stream(stream))
    return out


def hierarchical_sum(a: torch.Tensor, out: torch.Tensor, stream=None) -> torch.Tensor:
    """out[0] += sum(a) with one f32 atomic per block (reference semantics)."""
    o = c_p(out.data_ptr())
    call("spmdb200_hierarchical_sum", *memref(a), o, o, c_i(0), c_i(a.shape[0]), _stream(stream))
    return out


KINDS = {"add": 0, "mul": 1, "max": 2, "min": 3, "and": 4, "or": 5, "xor": 6}


def reduce(kind: str, a: torch.Tensor, init, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
           stream=None) -> torch.Tensor:
    """out[0] = init (+) a[0] (+) ... for an spmd.reduce kind (f32: add/mul/max/min; i32: all seven)."""
    n = a.shape[0]
    out = torch.empty(1, dtype=a.dtype, device=a.device) if out is None else out
    ws = sum_workspace(n, a.device) if ws is None else ws
    o = c_p(out.data_ptr())
    common = (*memref(a), o, o, c_i(0), c_i(n))
    if a.dtype == torch.float32:
        call("spmdb200_reduce_f32", ctypes.c_int(KINDS[kind]), *common, ctypes.c_float(init), c_p(ws.data_ptr()),
             ctypes.c_size_t(ws.numel()), _stream(stream))
    elif a.dtype == torch.int32:
        call("spmdb200_reduce_i32", ctypes.c_int(KINDS[kind]), *common, ctypes.c_int32(init), c_p(ws.data_ptr()),
             ctypes.c_size_t(ws.numel()), _stream(stream))
    else:
        raise TypeError("reduce takes float32 or int32 tensors")
    return out


def jacobi_workspace(device=None) -> torch.Tensor:
    return torch.zeros(int(lib().spmdb200_jacobi_workspace_bytes()), dtype=torch.uint8, device=device or "cuda")


def workspace_status(ws: torch.Tensor, stream=None) -> None:
    """Synchronises and raises SpmdError if the run left a device-side timeout."""
    call("spmdb200_workspace_status", c_p(ws.data_ptr()), _stream(stream))


def _jacobi(entry: str, u: torch.Tensor, v: torch.Tensor, sweeps: int, res_every: int,
            ws: torch.Tensor | None, res: torch.Tensor | None, check: bool, stream):
    ws = jacobi_workspace(u.device) if ws is None else ws
    nres = sweeps // res_every if res_every > 0 else 0
    if res is None and nres > 0:
        res = torch.zeros(nres, dtype=torch.float64, device=u.device)
    rp = c_p(res.data_ptr()) if res is not None else c_p(0)
    call(entry, *memref(u), *memref(v), c_i(sweeps), c_i(res_every), rp, c_p(ws.data_ptr()),
         ctypes.c_size_t(ws.numel()), _stream(stream))
    if check:
        workspace_status(ws, stream)
    return (u if sweeps % 2 == 0 else v), res


def jacobi2d(u: torch.Tensor, v: torch.Tensor, sweeps: int, res_every: int = 0, ws=None, res=None,
             check: bool = True, stream=None):
    """`sweeps` 5-point sweeps ping-ponging u -> v -> u ...; returns (final grid, residuals)."""
    return _jacobi("spmdb200_jacobi2d", u, v, sweeps, res_every, ws, res, check, stream)


def jacobi3d(u: torch.Tensor, v: torch.Tensor, sweeps: int, res_every: int = 0, ws=None, res=None,
             check: bool = True, stream=None):
    """`sweeps` 7-point sweeps ping-ponging u -> v -> u ...; returns (final grid, residuals)."""
    return _jacobi("spmdb200_jacobi3d", u, v, sweeps, res_every, ws, res, check, stream)


# ---- training-step operators ---------------------------------------------------
# They take f32, f16 and bf16 tensors, run on the tensors' own device (current or
# not) and on its current stream unless `stream` says otherwise.  They record no
# autograd graph: gradients are what the *_backward entry returns.  A given tensor
# that a call writes has its version counter raised, so that autograd refuses a
# graph that saved it before; adamw raises those of parameters and copies, which
# graphs hold, and not its states' (the replay of a captured call raises none).
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_E4M3 = torch.float8_e4m3fn
STATE_BLOCK = 256  # elements that share one scale of an 8-bit optimizer state
HELD_COLUMNS = 49145  # of the longest rows for which layer_norm takes no workspace


def _elsewhere(dev: int, stream) -> bool:
    """Whether a call has to enter a stream or device first (_at)."""
    if dev < 0:
        raise ValueError("device entries take CUDA tensors")
    return stream is not None or dev != torch._C._cuda_getDevice()


def _at(dev: int, stream):
    """Context in which launches and allocations belong to `stream`, or to the
    current stream of device `dev`."""
    if stream is None:
        return torch.cuda.device(dev)
    if stream.device_index != dev:
        raise ValueError(f"the stream belongs to cuda:{stream.device_index}, the tensors to cuda:{dev}")
    return torch.cuda.stream(stream)


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


_raise_versions = torch.autograd.graph.increment_version


def _ptr(a: array) -> int:
    """Address of a host array, which the caller keeps until the call is over."""
    return a.buffer_info()[0]


def _norm_operand(name: str, t: torch.Tensor, shape, dev: int, dtype=None) -> None:
    if t.get_device() != dev:
        raise ValueError(f"layer_norm: {name} is not on x's device")
    if t.shape != shape:
        raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if (t.dtype != dtype) if dtype is not None else (t.dtype not in _TYPES):
        raise TypeError(f"layer_norm: {name} has dtype {t.dtype}")


def _norm_vector(name: str, t: torch.Tensor, shape, dev: int, dtype=None) -> None:
    _norm_operand(name, t, shape, dev, dtype)
    if not t.is_contiguous():
        raise ValueError(f"layer_norm: {name} must be contiguous")


def _norm_rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """A view of rank 1-3 (leading dimensions merged where the rank is higher)."""
    if t.dim() <= 3:
        return t
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        raise ValueError(f"layer_norm: the leading dimensions of {name} do not merge into rows") from None


def _norm_types(x: torch.Tensor, y: torch.dtype) -> None:
    if x.dtype not in _TYPES or y not in _TYPES:
        raise TypeError(f"layer_norm: dtypes {x.dtype}, {y}")
    if x.dtype != y and x.dtype != torch.float32 and y != torch.float32:
        raise TypeError(f"layer_norm: {x.dtype} and {y}: equal, or one of them float32")


def _plain(**views: torch.Tensor) -> None:
    """Refuses views that torch negates lazily (the imaginary part of a conjugate): their memory holds other values."""
    for name, t in views.items():
        if t.is_neg():
            raise ValueError(f"layer_norm: {name} is negated lazily (resolve_neg gives its values)")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
               stats: bool = True, ws: torch.Tensor | None = None, stream=None):
    """(out, mean, rstd): layer norm over the last dimension, out = (x - mean) *
    rstd * weight + bias.  x is a strided view, of rank 1 to 3 or with leading
    dimensions that merge into rows; out has `dtype` (default
    x's; one of the two may be float32) and may be x itself.  mean and rstd
    (float32, x's leading shape) are what layer_norm_backward takes; stats=False
    leaves them out (None).  Rows of more than HELD_COLUMNS elements use a workspace of
    layer_norm_workspace(rows, cols, backward=False)."""
    dev = x.get_device()
    if _elsewhere(dev, stream):
        with _at(dev, stream):
            return layer_norm(x, weight, bias, eps, dtype, out, stats, ws)
    shape = x.shape
    if not shape:
        raise ValueError("layer_norm: x needs a dimension to normalise over")
    given = out is not None
    if given:
        _norm_operand("out", out, shape, dev, dtype)
    else:
        out = torch.empty(shape, dtype=dtype or x.dtype, device=x.device)
    _norm_types(x, out.dtype)
    w = b = m = r = mean = rstd = None
    wtype = 0
    if weight is not None:
        _norm_vector("weight", weight, shape[-1:], dev)
        w, wtype = weight.data_ptr(), _TYPES[weight.dtype]
    if bias is not None:
        _norm_vector("bias", bias, shape[-1:], dev, None if weight is None else weight.dtype)
        b, wtype = bias.data_ptr(), _TYPES[bias.dtype]
    if stats:
        mean = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        m, r = mean.data_ptr(), rstd.data_ptr()
    xv, ov = _norm_rows("x", x), _norm_rows("out", out)
    rank, room, room_bytes = xv.dim(), None, 0
    if ws is not None or shape[-1] > HELD_COLUMNS:
        ws = _norm_room(ws, math.prod(shape[:-1]), shape[-1], x, False)
        room, room_bytes = ws.data_ptr(), ws.nbytes
    xs, ys = xv.stride(), ov.stride()
    if xs[-1] != 1 or ys[-1] != 1:  # a negated view's columns are spread
        _plain(x=x, out=out)
    dims = array("q", (*xv.shape, *xs, *ys))
    at = _ptr(dims)
    call("spmdb200_layer_norm", rank, at, xv.data_ptr(), _TYPES[x.dtype], at + 8 * rank, ov.data_ptr(),
         _TYPES[out.dtype], at + 16 * rank, w, b, wtype, eps, m, r, room, room_bytes, _raw_stream(dev))
    if given:
        _raise_versions(out)
    return out, mean, rstd


def layer_norm_workspace(rows: int, cols: int, device=None, backward: bool = True) -> torch.Tensor:
    """Workspace for layer_norm_backward, or for layer_norm (contents irrelevant,
    reusable; calls that share it must not overlap on the GPU)."""
    size = lib().spmdb200_layer_norm_workspace_bytes if backward else lib().spmdb200_layer_norm_forward_workspace_bytes
    return torch.empty(size(rows, cols), dtype=torch.uint8, device=device or "cuda")


def _norm_room(ws: torch.Tensor | None, rows: int, cols: int, x: torch.Tensor, backward: bool) -> torch.Tensor:
    if ws is None:
        return layer_norm_workspace(rows, cols, x.device, backward)
    if ws.get_device() != x.get_device() or not ws.is_contiguous():
        raise ValueError("layer_norm: ws is a contiguous tensor on x's device")
    return ws


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None, wgrad: bool | None = None, dx: torch.Tensor | None = None,
                        dweight: torch.Tensor | None = None, dbias: torch.Tensor | None = None,
                        ws: torch.Tensor | None = None, stream=None):
    """(dx, dweight, dbias) of layer_norm from dy and its saved mean and rstd.
    dx has x's dtype and may be dy or x itself; dweight and dbias have weight's
    dtype (float32 without a weight) unless tensors are given.  wgrad=False
    leaves both out (None), the default without a weight."""
    dev = x.get_device()
    if _elsewhere(dev, stream):
        with _at(dev, stream):
            return layer_norm_backward(dy, x, mean, rstd, weight, wgrad, dx, dweight, dbias, ws)
    shape = x.shape
    if not shape:
        raise ValueError("layer_norm: x needs a dimension to normalise over")
    _norm_operand("dy", dy, shape, dev)
    _norm_types(x, dy.dtype)
    _norm_vector("mean", mean, shape[:-1], dev, torch.float32)
    _norm_vector("rstd", rstd, shape[:-1], dev, torch.float32)
    written = [t for t in (dx, dweight, dbias) if t is not None]
    w = dw = db = None
    wtype = dtype = 0
    if weight is not None:
        _norm_vector("weight", weight, shape[-1:], dev)
        w, wtype = weight.data_ptr(), _TYPES[weight.dtype]
    if wgrad is None:
        wgrad = weight is not None or dweight is not None or dbias is not None
    if wgrad:
        given = dweight if dweight is not None else dbias if dbias is not None else weight
        kind = torch.float32 if given is None else given.dtype
        dweight = torch.empty(shape[-1:], dtype=kind, device=x.device) if dweight is None else dweight
        dbias = torch.empty(shape[-1:], dtype=kind, device=x.device) if dbias is None else dbias
        _norm_vector("dweight", dweight, shape[-1:], dev)
        _norm_vector("dbias", dbias, shape[-1:], dev, dweight.dtype)
        dw, db, dtype = dweight.data_ptr(), dbias.data_ptr(), _TYPES[dweight.dtype]
    elif dweight is not None or dbias is not None:
        raise ValueError("layer_norm: dweight or dbias given with wgrad=False")
    if dx is None:
        dx = torch.empty(shape, dtype=x.dtype, device=x.device)
    else:
        _norm_operand("dx", dx, shape, dev, x.dtype)
    gv, xv, dv = _norm_rows("dy", dy), _norm_rows("x", x), _norm_rows("dx", dx)
    ws = _norm_room(ws, mean.numel(), shape[-1], x, True)
    rank = xv.dim()
    gs, xs, ds = gv.stride(), xv.stride(), dv.stride()
    if gs[-1] != 1 or xs[-1] != 1 or ds[-1] != 1:  # a negated view's columns are spread
        _plain(dy=dy, x=x, dx=dx)
    dims = array("q", (*xv.shape, *gs, *xs, *ds))
    at = _ptr(dims)
    call("spmdb200_layer_norm_backward", rank, at, gv.data_ptr(), _TYPES[dy.dtype], at + 8 * rank, xv.data_ptr(),
         _TYPES[x.dtype], at + 16 * rank, mean.data_ptr(), rstd.data_ptr(), w, wtype, dv.data_ptr(), at + 24 * rank, dw,
         db, dtype, ws.data_ptr(), ws.nbytes, _raw_stream(dev))
    if written:
        _raise_versions(written)
    return dx, dweight, dbias


def _read_list(*args):
    """_tensor_lists.read, which takes this function's place at its first use:
    nothing but lists of tensors needs the module, which belongs to one torch."""
    global _read_list, _written
    try:
        from ._tensor_lists import read, written
    except ImportError as e:
        raise ImportError("lists of tensors need _tensor_lists.so, built for this torch by "
                          f"`python spmd-dialect_b200/build.py`: {e}") from e
    _read_list, _written = read, written
    return read(*args)


def _kinds(*dtypes: torch.dtype) -> int:
    """Allowed dtypes of a list, as _tensor_lists.read takes them."""
    return sum(1 << (3 if d == _E4M3 else _TYPES[d]) for d in dtypes)


_ANY_FLOAT, _ONLY_F32, _ONLY_E4M3 = _kinds(*_TYPES), _kinds(torch.float32), _kinds(_E4M3)
_COPIES = _kinds(torch.float16, torch.bfloat16) | 256  # an entry may be None


def grad_norm(grads, max_norm: float | None = None, ws: torch.Tensor | None = None, stream=None):
    """(norm, scale): the 2-norm over every element of a list of tensors, and
    min(1, max_norm / norm) (None without max_norm; NaN when the norm is not
    finite), as float32 tensors of one element on the device.  adamw takes
    scale as its grad_scale, with no read by the host in between."""
    grads = list(grads)
    dev = grads[0].get_device() if grads else torch.cuda.current_device()
    if _elsewhere(dev, stream):
        with _at(dev, stream):
            return grad_norm(grads, max_norm, ws)
    ptrs, sizes, types = _read_list("grad_norm", grads, dev, _ANY_FLOAT, None)
    if ws is None:
        ws = torch.empty(lib().spmdb200_grad_norm_workspace_bytes(len(grads)), dtype=torch.uint8, device=f"cuda:{dev}")
    elif ws.get_device() != dev or not ws.is_contiguous():
        raise ValueError("grad_norm: ws is a contiguous tensor on the gradients' device")
    norm = torch.empty(1, dtype=torch.float32, device=ws.device)
    scale = None if max_norm is None else torch.empty_like(norm)
    call("spmdb200_grad_norm", len(grads), ptrs, sizes, types, 0.0 if max_norm is None else max_norm, norm.data_ptr(),
         None if scale is None else scale.data_ptr(), ws.data_ptr(), ws.nbytes, _raw_stream(dev))
    return norm, scale


def adamw_state(params, bits: int = 32) -> dict:
    """Zeroed states for adamw, as its keyword arguments: exp_avg and exp_avg_sq
    (float32, or float8_e4m3fn codes for bits=8) and for bits=8 their scales."""
    if bits not in (8, 32):
        raise ValueError("adamw: states have 8 or 32 bits")
    params, kind = list(params), torch.float32 if bits == 32 else _E4M3
    names = ["exp_avg", "exp_avg_sq"]
    state = {n: [torch.zeros(p.shape, dtype=kind, device=p.device) for p in params] for n in names}
    if bits == 8:
        for n in names:
            state[n + "_scales"] = [torch.zeros(-(-p.numel() // STATE_BLOCK), dtype=torch.float32, device=p.device)
                                    for p in params]
    return state


def _scalar(name: str, t: torch.Tensor, dev: int, dtype: torch.dtype) -> int:
    if t.get_device() != dev or t.dtype != dtype or t.numel() != 1:
        raise ValueError(f"adamw: {name} is one {dtype} element on the parameters' device")
    return t.data_ptr()


def adamw(params, grads, exp_avg, exp_avg_sq, *, step, lr, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01,
          exp_avg_scales=None, exp_avg_sq_scales=None, copies=None, grad_scale: torch.Tensor | None = None,
          stream=None):
    """One AdamW step over lists of contiguous tensors, in place; returns params.

    params and grads are float32, float16 or bfloat16, independently.  States
    hold as many elements as their parameter: float32, or float8_e4m3fn with
    their `*_scales` (adamw_state makes either).  copies: per parameter a
    float16 / bfloat16 tensor that receives the new value too, or None.
    weight_decay: a number, or one per parameter.  step (from 1) and lr are
    numbers, or one-element device tensors (int64, float32) that a captured
    step reads anew at each replay.  grad_scale multiplies every gradient; when
    it is NaN or infinite nothing is changed."""
    params, grads, exp_avg, exp_avg_sq = list(params), list(grads), list(exp_avg), list(exp_avg_sq)
    n = len(params)
    if not n:
        if grads or exp_avg or exp_avg_sq:
            raise ValueError("adamw: no parameters for the tensors given")
        return params
    dev = params[0].get_device()
    if _elsewhere(dev, stream):
        with _at(dev, stream):
            return adamw(params, grads, exp_avg, exp_avg_sq, step=step, lr=lr, betas=betas, eps=eps,
                         weight_decay=weight_decay, exp_avg_scales=exp_avg_scales, exp_avg_sq_scales=exp_avg_sq_scales,
                         copies=copies, grad_scale=grad_scale)
    bits = 8 if exp_avg_scales is not None or exp_avg_sq_scales is not None else 32
    state = _ONLY_F32 if bits == 32 else _ONLY_E4M3
    p, sizes, p_types = _read_list("adamw: params", params, dev, _ANY_FLOAT, None)
    g, _, g_types = _read_list("adamw: grads", grads, dev, _ANY_FLOAT, params)
    (m, m_sizes, _), (v, v_sizes, _) = (_read_list("adamw: " + name, ts, dev, state, None) for name, ts in (
        ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)))
    if m_sizes != sizes or v_sizes != sizes:
        raise ValueError("adamw: exp_avg and exp_avg_sq must have the parameters' sizes")
    m_scales = v_scales = c = c_types = None
    if bits == 8:
        blocks = array("q", [-(-k // STATE_BLOCK) for k in array("q", sizes)]).tobytes()
        (m_scales, m_blocks, _), (v_scales, v_blocks, _) = (
            _read_list("adamw: scales", [] if ts is None else list(ts), dev, _ONLY_F32, None)
            for ts in (exp_avg_scales, exp_avg_sq_scales))
        if m_blocks != blocks or v_blocks != blocks:
            raise ValueError(f"adamw: 8-bit states need one scale per {STATE_BLOCK} elements of each parameter")
    if copies is not None:
        copies = list(copies)
        c, _, c_types = _read_list("adamw: copies", copies, dev, _COPIES, params)
    decay = array("d", weight_decay) if hasattr(weight_decay, "__len__") else array("d", [weight_decay]) * n
    if len(decay) != n:
        raise ValueError("adamw: weight_decay is a number or one per parameter")
    lr_dev = step_dev = factor = None
    if isinstance(lr, torch.Tensor):
        lr, lr_dev = 0.0, _scalar("lr", lr, dev, torch.float32)
    if isinstance(step, torch.Tensor):
        step, step_dev = 1, _scalar("step", step, dev, torch.int64)
    if grad_scale is not None:
        factor = _scalar("grad_scale", grad_scale, dev, torch.float32)
    call("spmdb200_adamw", n, p, p_types, g, g_types, sizes, m, v, bits, m_scales, v_scales, c, c_types, _ptr(decay), lr,
         lr_dev, betas[0], betas[1], eps, step, step_dev, factor, _raw_stream(dev))
    _written(params, copies)
    return params
