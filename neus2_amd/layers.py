"""Layers of any width, beside the 64-wide FullyFusedMLP, and the clipping in front of the optimiser: linear layers with bias,
activation and residual, layer norm, and the norm over many tensors' gradients.

Matrices are row-per-sample tensors [N, C] in fp16 or bf16 (layer norm: also fp32) with any row stride; a layer's parameters are
one flat vector, as tcnn's networks have them (the reference reaches networks of other widths through the same create_network,
nerf_network.h:57 and :65).  As in tcnn_api torch is used for device memory and streams only; each call takes its workspace
from torch's allocator, so calls on several streams and in several graphs do not share one."""
import ctypes as C

import torch

from . import capi
from .capi import GRAD_IGNORE, GRAD_OVERWRITE, N2Error, check
from .tcnn_api import _address, _raw_stream, _stream_address

DTYPES = {torch.float16: capi.DTYPE_F16, torch.bfloat16: capi.DTYPE_BF16, torch.float32: capi.DTYPE_F32}
ACTIVATIONS = {"None": capi.ACTIVATION_NONE, "ReLU": capi.ACTIVATION_RELU, "SiLU": capi.ACTIVATION_SILU, "GELU": capi.ACTIVATION_GELU}


# not part of torch's public interface: where a torch does without it, the public call serves (which looks first whether CUDA is there, 0.3 us)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _check_device(t, what):
    """The current device's index, which has to be the tensor's."""
    device = t.get_device()
    if device < 0:
        raise N2Error(f"{what} must be a CUDA tensor")
    if device != _current_device():
        raise N2Error(f"{what} is on cuda:{device}, the current device is cuda:{_current_device()}")
    return device


def _stream_of(device):
    return _stream_address() if _raw_stream is None else _raw_stream(device)


def _matrix(t, dtype, device, rows, width, what):
    """The row stride of a [rows, width] tensor (rows None: any)."""
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 2 or shape[1] != width or (rows is not None and shape[0] != rows):
        raise N2Error(f"{what} must be a {dtype} tensor [{'N' if rows is None else rows}, {width}], got {t.dtype} {tuple(shape)}")
    if t.get_device() != device:
        _check_device(t, what)
    rows = shape[0]
    if rows >= 1 << 31:
        raise N2Error(f"{what} has {rows} rows, 2^31 - 1 are the most")
    if rows == 0:
        return width
    stride, inner = t.stride()
    if (inner != 1 and width > 1) or (stride < width and rows > 1):
        raise N2Error(f"{what} must have its rows' values side by side and its rows apart, got strides {t.stride()}")
    return stride if stride > width else width


def _vector(t, dtype, n, what):
    _check_device(t, what)
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise N2Error(f"{what} must be a contiguous {dtype} tensor of {n} elements, got {t.dtype} {tuple(t.shape)}")


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


class Linear:
    """y = act(x W^T + b) + residual.  Parameters: [W row-major [out, in] | b [out]] in one vector."""

    def __init__(self, n_input_dims, n_output_dims, activation="None", bias=True, dtype=torch.float16):
        if activation not in ACTIVATIONS:
            raise N2Error(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise N2Error(f"linear layers are fp16 or bf16, got {dtype}")
        if not (1 <= n_input_dims <= 65536 and 1 <= n_output_dims <= 65536):
            raise N2Error(f"widths {n_input_dims}, {n_output_dims} outside [1, 65536]")
        self.n_input_dims, self.n_output_dims, self.activation, self.bias, self.dtype = n_input_dims, n_output_dims, activation, bool(bias), dtype
        self._kinds = (DTYPES[dtype], ACTIVATIONS[activation])
        self._params = self._grads = None

    def n_params(self):
        return self.n_output_dims * (self.n_input_dims + self.bias)

    def input_width(self):
        return self.n_input_dims

    def output_width(self):
        return self.n_output_dims

    padded_output_width = output_width

    def set_params(self, params, gradients=None):
        """params / gradients: vectors of n_params elements in the layer's type (kept alive by this object)."""
        for t in (params, gradients):
            if t is not None:
                _vector(t, self.dtype, self.n_params(), "linear params/gradients")
        self._params, self._grads = params, gradients
        self._at, self._grads_at = self._parts(params), self._parts(gradients)

    def _parts(self, t):
        """Addresses of the weights and the bias in a parameter vector."""
        if t is None:
            return None, None
        return t.data_ptr(), t.data_ptr() + t.element_size() * self.n_output_dims * self.n_input_dims if self.bias else None

    def _ready(self):
        if self._params is None:
            raise N2Error("linear layer: call set_params first")
        return _check_device(self._params, "linear params")

    def forward(self, x, residual=None, want_pre_activation=False, out=None):
        """x [N, in]; residual [N, out] or None.  Returns (y [N, out], z [N, out] or None): z = x W^T + b is what backward of an
        activation takes.  out may be the residual itself."""
        device = self._ready()
        i, o, dtype = self.n_input_dims, self.n_output_dims, self.dtype
        x_stride, n = _matrix(x, dtype, device, None, i, "linear input"), x.shape[0]
        r_stride = o if residual is None else _matrix(residual, dtype, device, n, o, "linear residual")
        y, y_stride = (x.new_empty((n, o)), o) if out is None else (out, _matrix(out, dtype, device, n, o, "linear output"))
        z = x.new_empty((n, o)) if want_pre_activation else None
        lib = capi.lib()
        nbytes = lib.n2_linear_forward_workspace_bytes(n, i, o)
        ws = _workspace(nbytes, x)
        w, b = self._at
        rc = lib.n2_linear_forward(_stream_of(device), *self._kinds, n, i, o, w, b, x.data_ptr(), x_stride, _address(residual), r_stride, y.data_ptr(), y_stride, _address(z), o, _address(ws),
                                   nbytes)
        if rc:
            check(rc, "n2_linear_forward")
        return y, z

    def backward(self, x, pre_activation, dL_dy, want_input_grad=True, mode=GRAD_OVERWRITE, out=None):
        """Gradients of the layer's parameters go into the vector of set_params (by mode); returns dL/dx [N, in] or None.
        pre_activation: what forward returned (None without an activation).  The residual's gradient is dL_dy."""
        device = self._ready()
        i, o, dtype = self.n_input_dims, self.n_output_dims, self.dtype
        x_stride, n = _matrix(x, dtype, device, None, i, "linear input"), x.shape[0]
        dy_stride = _matrix(dL_dy, dtype, device, n, o, "dL_dy")
        z_stride = o
        if self.activation == "None":
            pre_activation = None
        elif pre_activation is None:
            raise N2Error(f"backward of {self.activation} needs the values before it: forward(want_pre_activation=True)")
        else:
            z_stride = _matrix(pre_activation, dtype, device, n, o, "pre_activation")
        if mode != GRAD_IGNORE and self._grads is None:
            raise N2Error("linear layer: set_params was given no gradients")
        dx, dx_stride = None, i
        if want_input_grad:
            dx, dx_stride = (x.new_empty((n, i)), i) if out is None else (out, _matrix(out, dtype, device, n, i, "dL_dx"))
        lib = capi.lib()
        nbytes = lib.n2_linear_backward_workspace_bytes(n, i, o)
        ws = _workspace(nbytes, x)
        dw, db = self._grads_at
        rc = lib.n2_linear_backward(_stream_of(device), *self._kinds, n, i, o, self._at[0], x.data_ptr(), x_stride, _address(pre_activation), z_stride, dL_dy.data_ptr(), dy_stride, _address(dx),
                                    dx_stride, dw, db, mode, _address(ws), nbytes)
        if rc:
            check(rc, "n2_linear_backward")
        return dx


class LayerNorm:
    """y = (x - mean) / sqrt(variance + epsilon) * scale + shift over each row.  Parameters: [scale | shift] in one vector, of the
    rows' type or fp32."""

    def __init__(self, n_dims, epsilon=1e-5, dtype=torch.float16, param_dtype=None):
        param_dtype = dtype if param_dtype is None else param_dtype
        if dtype not in DTYPES or param_dtype not in (dtype, torch.float32):
            raise N2Error(f"layer norm: rows of {dtype} with parameters of {param_dtype}")
        if not 1 <= n_dims <= 16384:
            raise N2Error(f"layer norm: width {n_dims} outside [1, 16384]")
        if not 0 < epsilon < float("inf"):
            raise N2Error(f"layer norm: epsilon {epsilon} must be positive")
        self.n_dims, self.epsilon, self.dtype, self.param_dtype = n_dims, epsilon, dtype, param_dtype
        self._kinds = (DTYPES[dtype], DTYPES[param_dtype])
        self._params = self._grads = None

    def n_params(self):
        return 2 * self.n_dims

    def input_width(self):
        return self.n_dims

    output_width = padded_output_width = input_width

    def set_params(self, params, gradients=None):
        """params / gradients: vectors of n_params elements (kept alive by this object)."""
        for t in (params, gradients):
            if t is not None:
                _vector(t, self.param_dtype, self.n_params(), "layer norm params/gradients")
        self._params, self._grads = params, gradients
        self._at, self._grads_at = self._parts(params), self._parts(gradients)

    def _ready(self):
        if self._params is None:
            raise N2Error("layer norm: call set_params first")
        return _check_device(self._params, "layer norm params")

    def _parts(self, t):
        return (None, None) if t is None else (t.data_ptr(), t.data_ptr() + t.element_size() * self.n_dims)

    def forward(self, x, want_ctx=False, out=None):
        """Returns (y, ctx): ctx = (mean, rstd), fp32 [N] each, is what backward takes (None unless asked for)."""
        device = self._ready()
        w, dtype = self.n_dims, self.dtype
        x_stride, n = _matrix(x, dtype, device, None, w, "layer norm input"), x.shape[0]
        y, y_stride = (x.new_empty((n, w)), w) if out is None else (out, _matrix(out, dtype, device, n, w, "layer norm output"))
        mean = rstd = ctx = None
        if want_ctx:
            ctx = mean, rstd = x.new_empty(n, dtype=torch.float32), x.new_empty(n, dtype=torch.float32)
        rc = capi.lib().n2_layer_norm_forward(_stream_of(device), *self._kinds, n, w, self.epsilon, *self._at, x.data_ptr(), x_stride, y.data_ptr(), y_stride, _address(mean), _address(rstd))
        if rc:
            check(rc, "n2_layer_norm_forward")
        return y, ctx

    def backward(self, ctx, x, dL_dy, dL_dskip=None, want_input_grad=True, mode=GRAD_OVERWRITE, out=None):
        """dL_dskip (or None): a gradient of x that is added to dL/dx, as a skip connection past the norm has it; out may be that tensor."""
        device = self._ready()
        if ctx is None:
            raise N2Error("layer norm: backward needs the ctx of forward(want_ctx=True)")
        w, dtype = self.n_dims, self.dtype
        x_stride, n = _matrix(x, dtype, device, None, w, "layer norm input"), x.shape[0]
        dy_stride = _matrix(dL_dy, dtype, device, n, w, "dL_dy")
        skip_stride = w if dL_dskip is None else _matrix(dL_dskip, dtype, device, n, w, "dL_dskip")
        mean, rstd = ctx
        _vector(mean, torch.float32, n, "mean")
        _vector(rstd, torch.float32, n, "rstd")
        if mode != GRAD_IGNORE and self._grads is None:
            raise N2Error("layer norm: set_params was given no gradients")
        if dL_dskip is not None and not want_input_grad:
            raise N2Error("layer norm: dL_dskip without dL/dx")
        dx, dx_stride = None, w
        if want_input_grad:
            dx, dx_stride = (x.new_empty((n, w)), w) if out is None else (out, _matrix(out, dtype, device, n, w, "dL_dx"))
        lib = capi.lib()
        nbytes = lib.n2_layer_norm_workspace_bytes(self._kinds[0], n, w) if mode != GRAD_IGNORE else 0
        ws = _workspace(nbytes, x)
        rc = lib.n2_layer_norm_backward(_stream_of(device), *self._kinds, n, w, self._at[0], x.data_ptr(), x_stride, mean.data_ptr(), rstd.data_ptr(), dL_dy.data_ptr(), dy_stride,
                                        _address(dL_dskip), skip_stride, _address(dx), dx_stride, *self._grads_at, mode, _address(ws), nbytes)
        if rc:
            check(rc, "n2_layer_norm_backward")
        return dx


class GradientClip:
    """The norm over the gradients of many tensors, and their scaling to at most a given norm, in front of an optimiser's step.

    gradients: tensors without gaps, fp16, bf16 and fp32 in any mixture, that do not overlap (kept alive here: every call reads what
    they hold then).  out: tensors of the same types and sizes for the clipped gradients; None clips in place.  The table of the tensors'
    addresses is this object's: calls on any stream may be under way when it is dropped, but a captured graph needs it alive."""

    def __init__(self, gradients, out=None):
        gradients = list(gradients)
        out = gradients if out is None else list(out)
        if len(out) != len(gradients):
            raise N2Error(f"{len(gradients)} gradients, {len(out)} outputs")
        tensors = (capi.GradientTensor * max(len(gradients), 1))()
        for i, (g, o) in enumerate(zip(gradients, out)):
            for t in (g, o):
                _check_device(t, f"gradient {i}")
                if t.dtype not in DTYPES or not t.is_contiguous():
                    raise N2Error(f"gradient {i} must be a contiguous fp16, bf16 or fp32 tensor")
            if o.dtype != g.dtype or o.shape != g.shape:
                raise N2Error(f"gradient {i} is {g.dtype} {tuple(g.shape)}, its output {o.dtype} {tuple(o.shape)}")
            tensors[i] = capi.GradientTensor(g.data_ptr(), o.data_ptr(), g.numel(), DTYPES[g.dtype])
        L = capi.lib()
        nbytes = L.n2_gradients_table_bytes(len(gradients), tensors)
        self._keep = (gradients, out)
        self._table = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        self._stream = _stream_of(_current_device())
        self._h = C.c_void_p()
        check(L.n2_gradients_create(self._stream, len(gradients), tensors, self._table.data_ptr(), nbytes, C.byref(self._h)), "n2_gradients_create")

    def __del__(self):
        try:
            if getattr(self, "_h", None) is not None and self._h.value:
                capi.lib().n2_gradients_destroy(self._h)
                self._h = C.c_void_p()
        except Exception:
            pass

    def _buffers(self):
        table = self._table
        stream = _stream_of(_check_device(table, "the gradients' table"))
        if stream != self._stream:  # (the table's memory goes to nobody else before this stream has read it)
            table.record_stream(torch.cuda.current_stream())
        return stream, table.new_empty((), dtype=torch.float32), table.new_empty(capi.GRADIENTS_WORKSPACE_BYTES)

    def norm(self, loss_scale=1.0):
        """sqrt(sum of squares) / loss_scale as a one-element device tensor (no host synchronisation)."""
        stream, norm, ws = self._buffers()
        check(capi.lib().n2_gradients_norm(self._h, stream, loss_scale, norm.data_ptr(), ws.data_ptr(), capi.GRADIENTS_WORKSPACE_BYTES), "n2_gradients_norm")
        return norm

    def clip(self, max_norm, loss_scale=1.0):
        """Multiplies the gradients by min(1, max_norm / (norm + 1e-6)); they keep their loss scale (Adam.step's, whose gradients
        are loss_scale times the loss's).  Returns the norm before, as norm() does."""
        stream, norm, ws = self._buffers()
        check(capi.lib().n2_gradients_clip(self._h, stream, max_norm, loss_scale, norm.data_ptr(), ws.data_ptr(), capi.GRADIENTS_WORKSPACE_BYTES), "n2_gradients_clip")
        return norm
