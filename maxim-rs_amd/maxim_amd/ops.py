"""ctypes binding of the operators on device tensors (include/maxim_ops.h):
LayerNorm and Dense, forward and backward, in fp32, fp16 or bf16.

Tensors are torch's, on the card; results and workspaces come from torch's
allocator and the kernels go to torch's current stream of that device, so the
calls mix with torch's own work and can be captured into its graphs (after
`ready()`, which loads the kernels). There is no CPU fallback. torch has to be
imported before the process first uses the executor, so that both share one
HIP runtime; otherwise the calls are refused.

Features are a tensor's last dimension, positions all the others (token
order, the default), or, with planar=True, features the first dimension and
positions the rest: the executor's [c][h][w]. Any strides will do that make
either the features or the positions contiguous; others are refused, not
copied. Results have x's memory order (Dense's y and z the residual's, where
there is one). The calls record no autograd graph: each forward call has a backward
call beside it, and tensors that require a gradient are refused while torch
records one (use torch.no_grad(), as an autograd.Function's methods do); so are
tensors that carry a forward-mode tangent.
"""

import ctypes as C

from . import plan as P
from .hip import _lib as _hip_lib

ACTS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "lrelu": 4, "sigmoid": 5}


class Mat(C.Structure):
    """mxh_mat"""
    _fields_ = [("data", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64), ("row_stride", C.c_int64),
                ("col_stride", C.c_int64), ("dtype", C.c_int32), ("reserved", C.c_int32)]


class Vec(C.Structure):
    """mxh_vec"""
    _fields_ = [("data", C.c_void_p), ("n", C.c_int64), ("dtype", C.c_int32), ("reserved", C.c_int32)]


_L = None
_torch = None
_forward_ad = None
_raw_stream = None
_types = {}


def _runtimes():
    """The HIP runtimes mapped into this process."""
    with open("/proc/self/maps") as f:
        return sorted({line.split()[-1] for line in f if "libamdhip64" in line})


def _lib():
    """The library with the operators' entry points declared."""
    global _L, _torch, _forward_ad, _raw_stream
    if _L is None:
        try:
            import torch  # before the library looks for a HIP runtime: torch's is the one to share
        except ImportError as e:
            raise P.MaximError("maxim_amd.ops works on torch tensors: %s" % e)
        if len(_runtimes()) > 1:
            # the executor has brought its own up; torch's tensors and streams are unknown to it
            raise P.MaximError("two HIP runtimes in the process (%s): import torch before the executor's first use"
                               % ", ".join(_runtimes()))
        L = _hip_lib()
        V, I, F, U = C.c_void_p, C.c_int, C.c_float, C.c_uint64
        M, N, B = C.POINTER(Mat), C.POINTER(Vec), C.POINTER(C.c_uint64)
        sig = {
            "mxh_ops_ready": [I],
            "mxh_layernorm": [I, V, M, N, N, F, M, V, V],
            "mxh_layernorm_backward": [I, V, M, M, N, V, V, M, M, N, N, V, U],
            "mxh_layernorm_backward_workspace": [M, B],
            "mxh_dense": [I, V, M, M, N, I, F, M, M, M, V, U],
            "mxh_dense_workspace": [M, M, M, B],
            "mxh_dense_backward": [I, V, M, M, M, M, I, F, M, M, N, V, U],
            "mxh_dense_backward_workspace": [M, M, M, I, M, M, N, B],
        }
        for name, args in sig.items():
            f = getattr(L, name)
            f.restype = I
            f.argtypes = args
        _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _torch, _forward_ad = torch, torch.autograd.forward_ad
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _L = L  # last: another thread that sees it sees the rest
    return _L


def _check(rc):
    if rc != 0:
        raise P.MaximError(P.last_error())


def _tensor(t, what, device):
    """The tensor's type code, or why it is refused."""
    try:
        code = _types.get(t.dtype)
        if code is not None and t.is_cuda and t.get_device() == device and not (
                t.requires_grad and _torch.is_grad_enabled()) and (
                _forward_ad._current_level < 0 or _forward_ad.unpack_dual(t).tangent is None):
            return code
    except AttributeError:
        raise P.MaximError("%s: not a tensor" % what)
    if not t.is_cuda:
        raise P.MaximError("%s: not on the card" % what)
    if t.get_device() != device:
        raise P.MaximError("%s: on another device than x" % what)
    if code is None:
        raise P.MaximError("%s: %s, not float32, float16 or bfloat16" % (what, t.dtype))
    if not (t.requires_grad and _torch.is_grad_enabled()):
        raise P.MaximError("%s carries a forward-mode tangent, which this call would drop" % what)
    raise P.MaximError("%s requires a gradient, which this call does not record: use torch.no_grad()" % what)


def _mat(t, what, device, planar):
    """A tensor as a matrix of positions and features."""
    code = _tensor(t, what, device)
    shape = t.shape
    if len(shape) != 2:
        if len(shape) < 2:
            raise P.MaximError("%s: %d dimensions, expected at least 2" % (what, len(shape)))
        c = shape[0] if planar else shape[-1]
        p = 1
        for d in shape[1:] if planar else shape[:-1]:
            p *= d
        flat = (c, p) if planar else (p, c)
        try:
            t = t.view(flat) if t.numel() else t.new_empty(flat)
        except RuntimeError:
            raise P.MaximError("%s: its positions have no one stride (shape %s, strides %s)"
                               % (what, tuple(shape), t.stride()))
        shape = t.shape
    a, b = shape
    sa, sb = t.stride()
    if planar:
        return Mat(t.data_ptr(), b, a, sb, sa, code, 0)
    return Mat(t.data_ptr(), a, b, sa, sb, code, 0)


def _vec(t, what, device):
    code = _tensor(t, what, device)
    if t.dim() != 1 or (t.stride(0) != 1 and t.shape[0] > 1):
        raise P.MaximError("%s: not a contiguous vector" % what)
    return Vec(t.data_ptr(), t.shape[0], code, 0)


def _device(x):
    _lib()
    if not isinstance(x, _torch.Tensor) or not x.is_cuda:
        raise P.MaximError("x: not a tensor on the card")
    return x.get_device()


def _stream(device):
    """torch's current stream of the device. (The raw lookup where torch has
    it: a tenth of a microsecond instead of more than one.)"""
    return _raw_stream(device) if _raw_stream else _torch.cuda.current_stream(device).cuda_stream


def _act(act):
    if act not in ACTS:
        raise P.MaximError("unknown activation %r (one of %s)" % (act, ", ".join(map(repr, ACTS))))
    return ACTS[act]


def _new(x, X, n, planar):
    """An uninitialised result of x's positions with n features, in x's memory
    order (X: x as a matrix): the tensor, and it as a matrix."""
    if n == X.cols and x.is_contiguous():
        t, by_rows = _torch.empty_like(x), planar
    else:
        rest = tuple(x.shape[1:] if planar else x.shape[:-1])
        # both strides 1, or a single position: the call's own order
        by_rows = planar if X.rows <= 1 or X.row_stride == X.col_stride == 1 else X.row_stride == 1
        t = x.new_empty((n,) + rest if by_rows else rest + (n,))
        if by_rows != planar:
            t = t.movedim(-1, 0) if planar else t.movedim(0, -1)
    return t, Mat(t.data_ptr(), X.rows, n, 1 if by_rows else n, X.rows if by_rows else 1, X.dtype, 0)


def _workspace(n, x):
    return x.new_empty(n, dtype=_torch.uint8) if n else None


def _written(out):
    """Tells autograd that a caller's tensor has new values (a result of the
    call's own has no history)."""
    if out is not None:
        _torch.autograd.graph.increment_version(out)


def _ptr(t):
    return None if t is None else t.data_ptr()


def ready(device=0):
    """mxh_ops_ready: loads the kernels (before the first capture)."""
    _check(_lib().mxh_ops_ready(device))


def layernorm(x, scale, bias=None, eps=1e-6, planar=False, stats=False, out=None):
    """mxh_layernorm: y of x's shape, or with stats (y, mean, rstd), the
    statistics fp32 with one value a position. out may be x."""
    d = _device(x)
    X = _mat(x, "x", d, planar)
    S = _vec(scale, "scale", d)
    B = None if bias is None else _vec(bias, "bias", d)
    y, Y = _new(x, X, X.cols, planar) if out is None else (out, X if out is x else _mat(out, "out", d, planar))
    mean = rstd = None
    if stats:
        shape = x.shape[1:] if planar else x.shape[:-1]
        mean = x.new_empty(shape, dtype=_torch.float32)
        rstd = _torch.empty_like(mean)
    _check(_L.mxh_layernorm(d, _stream(d), X, S, B, eps, Y, _ptr(mean), _ptr(rstd)))
    _written(out)
    return (y, mean, rstd) if stats else y


def layernorm_backward(dy, x, scale, mean, rstd, add=None, planar=False, dx=True, params=True, out=None):
    """mxh_layernorm_backward: (dx, dscale, dbias), None where dx or params is
    off. `add` is added to dx: the gradient that reaches x past the LayerNorm.
    out, for dx, may be dy or add."""
    d = _device(x)
    X = _mat(x, "x", d, planar)
    DY = _mat(dy, "dy", d, planar)
    S = _vec(scale, "scale", d)
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if _tensor(t, what, d) != 0 or t.numel() != X.rows or not t.is_contiguous():
            raise P.MaximError("%s: not a contiguous fp32 value for each position" % what)
    A = None if add is None else _mat(add, "add", d, planar)
    gx = DX = ds = db = DS = DB = ws = None
    if dx:
        if out is None:
            gx, DX = _new(x, X, X.cols, planar)
        else:
            gx, DX = out, DY if out is dy else A if out is add else _mat(out, "out", d, planar)
    elif out is not None:
        raise P.MaximError("out without dx")
    n = 0
    if params:
        ds = scale.new_empty(S.n)
        db = _torch.empty_like(ds)
        DS, DB = Vec(ds.data_ptr(), S.n, S.dtype, 0), Vec(db.data_ptr(), S.n, S.dtype, 0)
        size = C.c_uint64()
        _check(_L.mxh_layernorm_backward_workspace(X, size))
        n = size.value
        ws = _workspace(n, x)
    _check(_L.mxh_layernorm_backward(d, _stream(d), DY, X, S, mean.data_ptr(), rstd.data_ptr(), A, DX, DS, DB,
                                     _ptr(ws), n))
    _written(out)
    return gx, ds, db


def dense(x, w, bias=None, act=None, slope=0.0, residual=None, planar=False, save=False, out=None):
    """mxh_dense: act(x w^T + bias) + residual for w [n][k] (a [k][n] kernel
    goes in as its .t()), or with save (y, z), z the pre-activation that
    dense_backward takes. out may be the residual."""
    d = _device(x)
    a = _act(act)
    X = _mat(x, "x", d, planar)
    W = _mat(w, "w", d, False)
    B = None if bias is None else _vec(bias, "bias", d)
    R = None if residual is None else _mat(residual, "residual", d, planar)
    like, Like = (x, X) if residual is None else (residual, R)
    y, Y = _new(like, Like, W.rows, planar) if out is None else (out, _mat(out, "out", d, planar))
    z, Z = _new(y, Y, W.rows, planar) if save else (None, None)
    size = C.c_uint64()
    _check(_L.mxh_dense_workspace(X, W, Y, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_dense(d, _stream(d), X, W, B, a, slope, R, Y, Z, _ptr(ws), size.value))
    _written(out)
    return (y, z) if save else y


def dense_backward(dy, x, w, z=None, act=None, slope=0.0, planar=False, dx=True, dw=True, db=True, db_dtype=None):
    """mxh_dense_backward: (dx, dw, db) of dense(x, w, bias, act, slope), None
    where one is off. db is of w's type or db_dtype (the bias's: w's or
    float32). A residual's gradient is dy itself."""
    d = _device(x)
    a = _act(act)
    X = _mat(x, "x", d, planar)
    DY = _mat(dy, "dy", d, planar)
    W = _mat(w, "w", d, False)
    Z = None if z is None else _mat(z, "z", d, planar)
    gx = gw = gb = DX = DW = DB = None
    if dx:
        gx, DX = _new(x, X, X.cols, planar)
    if dw:
        # in w's own memory order
        gw = w.new_empty(w.shape) if W.col_stride == 1 else w.new_empty((W.cols, W.rows)).t()
        DW = (Mat(gw.data_ptr(), W.rows, W.cols, W.cols, 1, W.dtype, 0) if W.col_stride == 1 else
              Mat(gw.data_ptr(), W.rows, W.cols, 1, W.rows, W.dtype, 0))
    if db:
        gb = w.new_empty(W.rows, dtype=db_dtype)
        DB = _vec(gb, "db", d)
    size = C.c_uint64()
    _check(_L.mxh_dense_backward_workspace(DY, X, W, a, DX, DW, DB, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_dense_backward(d, _stream(d), DY, X, W, Z, a, slope, DX, DW, DB, _ptr(ws), size.value))
    return gx, gw, gb
