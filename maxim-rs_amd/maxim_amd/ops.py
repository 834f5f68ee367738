"""ctypes binding of the operators on device tensors (include/maxim_ops.h,
include/maxim_block_ops.h): LayerNorm, Dense and gated Dense, forward and
backward, in fp32, fp16 or bf16; the gradients' norm and clipping; 4-bit blocks
and the Dense of them.

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


class Mx4Mat(C.Structure):
    """mxh_mx4"""
    _fields_ = [("codes", C.c_void_p), ("scales", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64)]


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
        Q = C.POINTER(Mx4Mat)
        sig = {
            "mxh_ops_ready": [I],
            "mxh_layernorm": [I, V, M, N, N, F, M, V, V],
            "mxh_layernorm_backward": [I, V, M, M, N, V, V, M, M, N, N, V, U],
            "mxh_layernorm_backward_workspace": [M, B],
            "mxh_dense": [I, V, M, M, N, I, F, M, M, M, V, U],
            "mxh_dense_workspace": [M, M, M, B],
            "mxh_dense_backward": [I, V, M, M, M, M, I, F, M, M, N, V, U],
            "mxh_dense_backward_workspace": [M, M, M, I, M, M, N, B],
            "mxh_gated": [I, V, M, M, N, I, F, M, M, V, U],
            "mxh_gated_workspace": [M, M, M, M, B],
            "mxh_gated_backward": [I, V, M, M, M, M, I, F, M, M, N, V, U],
            "mxh_gated_backward_workspace": [M, M, M, M, M, N, B],
            "mxh_grad_norm": [I, V, N, C.c_int64, V, V, U],
            "mxh_grad_norm_workspace": [N, C.c_int64, B],
            "mxh_grad_clip": [I, V, N, N, C.c_int64, F, V, V, U],
            "mxh_grad_clip_by": [I, V, N, N, C.c_int64, F, V],
            "mxh_mx4_size": [C.c_int64, C.c_int64, B, B],
            "mxh_mx4_quantize": [I, V, M, Q],
            "mxh_mx4_dequantize": [I, V, Q, M],
            "mxh_mx4_dense": [I, V, M, Q, N, I, F, M, M, V, U],
            "mxh_mx4_dense_workspace": [M, Q, M, M, B],
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


def _either(X):
    """Whether a matrix lies in both orders: both strides 1, or one position."""
    return X.rows <= 1 or X.row_stride == X.col_stride == 1


def _new(x, X, n, planar, other=None):
    """An uninitialised result of x's positions with n features, in x's memory
    order (X: x as a matrix), or where x lies in both the other matrix's: the
    tensor, and it as a matrix."""
    if n == X.cols and x.is_contiguous():
        t, by_rows = _torch.empty_like(x), planar
    else:
        rest = tuple(x.shape[1:] if planar else x.shape[:-1])
        order = other if other is not None and _either(X) else X
        by_rows = planar if _either(order) else order.row_stride == 1  # the call's own order if both lie in both
        t = x.new_empty((n,) + rest if by_rows else rest + (n,))
        if by_rows != planar:
            t = t.movedim(-1, 0) if planar else t.movedim(0, -1)
    return t, Mat(t.data_ptr(), X.rows, n, 1 if by_rows else n, X.rows if by_rows else 1, X.dtype, 0)


def _like_weight(w, W):
    """An uninitialised result of a weight's shape, in its memory order."""
    if W.col_stride == 1:
        t = w.new_empty(w.shape)
        return t, Mat(t.data_ptr(), W.rows, W.cols, W.cols, 1, W.dtype, 0)
    t = w.new_empty((W.cols, W.rows)).t()
    return t, Mat(t.data_ptr(), W.rows, W.cols, 1, W.rows, W.dtype, 0)


def _workspace(n, x):
    return x.new_empty(n, dtype=_torch.uint8) if n else None


def _written(out):
    """Tells autograd that a caller's tensor, or each of a list, has new values
    (a result of the call's own has no history)."""
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
        gw, DW = _like_weight(w, W)
    if db:
        gb = w.new_empty(W.rows, dtype=db_dtype)
        DB = _vec(gb, "db", d)
    size = C.c_uint64()
    _check(_L.mxh_dense_backward_workspace(DY, X, W, a, DX, DW, DB, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_dense_backward(d, _stream(d), DY, X, W, Z, a, slope, DX, DW, DB, _ptr(ws), size.value))
    return gx, gw, gb


def gated(x, w, bias=None, act="silu", slope=0.0, planar=False, save=False, out=None):
    """mxh_gated: act(a) * c for (a | c) = x w^T + bias, w [2 n][k] with the
    gate's n rows first, or with save (y, z), z = (a | c) for gated_backward."""
    d = _device(x)
    f = _act(act)
    X = _mat(x, "x", d, planar)
    W = _mat(w, "w", d, False)
    B = None if bias is None else _vec(bias, "bias", d)
    y, Y = _new(x, X, W.rows // 2, planar) if out is None else (out, _mat(out, "out", d, planar))
    z, Z = _new(y, Y, W.rows, planar, X) if save else (None, None)  # a y of one feature has both orders
    size = C.c_uint64()
    _check(_L.mxh_gated_workspace(X, W, Y, Z, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_gated(d, _stream(d), X, W, B, f, slope, Y, Z, _ptr(ws), size.value))
    _written(out)
    return (y, z) if save else y


def gated_backward(dy, x, w, z, act="silu", slope=0.0, planar=False, dx=True, dw=True, db=True, db_dtype=None):
    """mxh_gated_backward: (dx, dw, db) of gated(x, w, bias, act, slope), None
    where one is off. db is of w's type or db_dtype (the bias's: w's or
    float32). In 16 bits the products take dz rounded to x's type, in fp16 scaled
    into its range."""
    d = _device(x)
    f = _act(act)
    X = _mat(x, "x", d, planar)
    DY = _mat(dy, "dy", d, planar)
    W = _mat(w, "w", d, False)
    Z = _mat(z, "z", d, planar)
    gx = gw = gb = DX = DW = DB = None
    if dx:
        gx, DX = _new(x, X, X.cols, planar)
    if dw:
        gw, DW = _like_weight(w, W)
    if db:
        gb = w.new_empty(W.rows, dtype=db_dtype)
        DB = _vec(gb, "db", d)
    size = C.c_uint64()
    _check(_L.mxh_gated_backward_workspace(DY, X, W, DX, DW, DB, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_gated_backward(d, _stream(d), DY, X, W, Z, f, slope, DX, DW, DB, _ptr(ws), size.value))
    return gx, gw, gb


def _filled(t, what):
    """The tensor's elements lie side by side, in whatever order."""
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            raise P.MaximError("%s: its elements do not fill its storage (shape %s, strides %s)"
                               % (what, tuple(t.shape), t.stride()))
        at *= size


def _list(tensors, what, device):
    """Tensors as an array of vectors of their elements. (Lists are long: the
    ordinary tensor's checks are here, _tensor has the others' and the words.)"""
    a = []
    plain = _forward_ad._current_level < 0
    try:
        for t in tensors:
            code = _types.get(t.dtype)
            if code is None or t.get_device() != device or t.requires_grad or not plain:
                code = _tensor(t, what, device)
            n = t.numel()
            if not t.is_contiguous() and n:
                _filled(t, what)
            a += (t.data_ptr(), n, code)  # a Vec's words, its type with the reserved half
    except P.MaximError as e:
        raise P.MaximError(str(e).replace(what, "%s[%d]" % (what, len(a) // 3), 1))
    except AttributeError:
        raise P.MaximError("%s[%d]: not a tensor" % (what, len(a) // 3))
    return (Vec * len(tensors)).from_buffer((C.c_int64 * len(a))(*a))


def _grads(grads):
    grads = list(grads)
    if not grads:
        raise P.MaximError("grads: no tensors")
    _lib()
    if not isinstance(grads[0], _torch.Tensor) or not grads[0].is_cuda:
        raise P.MaximError("grads[0]: not a tensor on the card")
    return grads, grads[0].get_device()


def _norm_workspace(a, like):
    size = C.c_uint64()
    _check(_L.mxh_grad_norm_workspace(a, len(a), size))
    return _workspace(size.value, like), size.value


def grad_norm(grads):
    """mxh_grad_norm: the 2-norm of all the tensors' elements together, an fp32
    tensor of no dimensions on their device."""
    grads, d = _grads(grads)
    a = _list(grads, "grads", d)
    norm = grads[0].new_empty((), dtype=_torch.float32)
    ws, n = _norm_workspace(a, grads[0])
    _check(_L.mxh_grad_norm(d, _stream(d), a, len(a), norm.data_ptr(), _ptr(ws), n))
    return norm


def clip_grads(grads, max_norm, norm=None, out=None):
    """mxh_grad_clip: scales the tensors in place, or into the tensors of out, by
    max_norm / N where their global norm N is larger than max_norm (and finite),
    and returns N. With norm (an fp32 tensor of one element, such as one added
    up over ranks) that is taken as N."""
    grads, d = _grads(grads)
    a = _list(grads, "grads", d)
    b = None
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise P.MaximError("out: %d tensors for %d gradients" % (len(out), len(grads)))
        b = _list(out, "out", d)
        for i, (g, o) in enumerate(zip(grads, out)):
            if not (g.is_same_size(o) and (g.is_contiguous() and o.is_contiguous() or g.stride() == o.stride())):
                raise P.MaximError("out[%d]: not its gradient's shape and strides" % i)
    if norm is None:
        norm = grads[0].new_empty((), dtype=_torch.float32)
        ws, n = _norm_workspace(a, grads[0])
        _check(_L.mxh_grad_clip(d, _stream(d), a, b, len(a), max_norm, norm.data_ptr(), _ptr(ws), n))
    else:
        if _tensor(norm, "norm", d) != 0 or norm.numel() != 1:
            raise P.MaximError("norm: not one fp32 value")
        _check(_L.mxh_grad_clip_by(d, _stream(d), a, b, len(a), max_norm, norm.data_ptr()))
    _written(grads if out is None else out)
    return norm


class Mx4:
    """A tensor in 4-bit blocks along its features (mxh_mx4): `codes` and
    `scales` (uint8, on the card), `shape` (positions, then features) and the
    `dtype` of the tensor that it was made from."""

    def __init__(self, data, code_bytes, rows, shape, dtype):
        self._data, self._code_bytes, self._rows = data, code_bytes, rows
        self.shape, self.dtype = shape, dtype

    codes = property(lambda self: self._data[:self._code_bytes])
    scales = property(lambda self: self._data[self._code_bytes:])

    def _mat(self):
        at = self._data.data_ptr()
        return Mx4Mat(at, at + self._code_bytes, self._rows, self.shape[-1])

    def plain(self):
        """(codes, scales) as [rows][features / 2 bytes] and [rows][blocks]
        tensors: the order in which others keep such blocks."""
        rows, cols = self._rows, self.shape[-1]
        tiles, groups, blocks = (cols + 255) // 256, (rows + 63) // 64, (cols + 31) // 32
        s = self.scales.view(groups, tiles, 4, 16, 4, 2).permute(0, 4, 3, 1, 5, 2).reshape(groups * 64, tiles * 8)
        return self.codes.view(rows, tiles * 128)[:, :(cols + 1) // 2], s[:rows, :blocks]


def mx4_quantize(x, planar=False):
    """mxh_mx4_quantize: x as an Mx4, in blocks along its features."""
    d = _device(x)
    X = _mat(x, "x", d, planar)
    codes, scales = C.c_uint64(), C.c_uint64()
    _check(_L.mxh_mx4_size(X.rows, X.cols, codes, scales))
    shape = tuple(x.shape[1:]) + (x.shape[0],) if planar else tuple(x.shape)
    # one allocation for both: codes are lines of 128 bytes
    q = Mx4(x.new_empty(codes.value + scales.value, dtype=_torch.uint8), codes.value, X.rows, shape, x.dtype)
    _check(_L.mxh_mx4_quantize(d, _stream(d), X, q._mat()))
    return q


def _mx4(q, what, device):
    if not isinstance(q, Mx4):
        raise P.MaximError("%s: not an Mx4" % what)
    if q._data.get_device() != device:
        raise P.MaximError("%s: on another device than x" % what)
    return q._mat()


def mx4_dequantize(q, dtype=None, planar=False):
    """mxh_mx4_dequantize: the values that an Mx4 stands for, as a tensor of
    dtype (the original's if None)."""
    _lib()
    if not isinstance(q, Mx4):
        raise P.MaximError("q: not an Mx4")
    d = q._data.get_device()
    m = q._mat()
    dtype = dtype or q.dtype
    y = q._data.new_empty((q.shape[-1],) + q.shape[:-1] if planar else q.shape, dtype=dtype)
    Y = (Mat(y.data_ptr(), m.rows, m.cols, 1, m.rows, 0, 0) if planar else
         Mat(y.data_ptr(), m.rows, m.cols, m.cols, 1, 0, 0))
    Y.dtype = _tensor(y, "y", d)
    _check(_L.mxh_mx4_dequantize(d, _stream(d), m, Y))
    return y


def mx4_dense(x, w, bias=None, act=None, slope=0.0, residual=None, planar=False, out=None):
    """mxh_mx4_dense: act(X W^T + bias) + residual with w an Mx4 of [n][k] and x
    taken to 4-bit blocks in the call. out may be the residual."""
    d = _device(x)
    a = _act(act)
    X = _mat(x, "x", d, planar)
    W = _mx4(w, "w", d)
    B = None if bias is None else _vec(bias, "bias", d)
    R = None if residual is None else _mat(residual, "residual", d, planar)
    like, Like = (x, X) if residual is None else (residual, R)
    y, Y = _new(like, Like, W.rows, planar) if out is None else (out, _mat(out, "out", d, planar))
    size = C.c_uint64()
    _check(_L.mxh_mx4_dense_workspace(X, W, R, Y, size))
    ws = _workspace(size.value, x)
    _check(_L.mxh_mx4_dense(d, _stream(d), X, W, B, a, slope, R, Y, _ptr(ws), size.value))
    _written(out)
    return y
