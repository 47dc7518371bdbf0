"""rusttorch_b200 — rusttorch-core's data-parallel tensor hot path on B200.

The Python surface mirrors rusttorch's PyO3 module (rusttorch-py/src/lib.rs):
the same function names, argument meaning and error behaviour (every failure
raises ValueError, here the RusttorchError subclass carrying the TensorError
variant).  The difference is where the data lives: a `Tensor` here is a
buffer in GPU memory (float32, unless a token operator says otherwise), and
every op is one call into librusttorch_cuda.so (see include/rusttorch_cuda.h).
Ops are asynchronous on the calling thread's stream; `to_numpy()` and the scalar reductions wait.
"""
from __future__ import annotations

import ctypes
from ctypes import c_double, c_void_p

import numpy as np

from . import _native
from ._native import F32, RusttorchError, check, lib

__all__ = [
    "Tensor", "TensorList", "RusttorchError", "version",
    "add", "sub", "mul", "div", "add_scalar", "mul_scalar", "add_mul_scalar",
    "fused_multiply_add", "add_simd", "mul_simd", "relu_simd", "mul_scalar_simd",
    "relu", "leaky_relu", "sigmoid", "tanh", "gelu", "swish", "elu", "selu", "mish",
    "softplus", "softsign", "softmax",
    "sum", "mean", "max", "min", "stats", "sum_dim", "mean_dim", "max_dim",
    "adam_update", "adamw_update", "sgd_update", "sgd_momentum_update",
    "add_broadcast", "sub_broadcast", "mul_broadcast", "div_broadcast",
    "nn_adam_step", "nn_sgd_step",
    "synchronize", "set_math_mode", "get_math_mode", "math_mode",
    "embedding", "embedding_backward", "softmax_cross_entropy", "softmax_cross_entropy_backward",
    "softmax_cross_entropy_grad", "adamw_update_multi", "adamw8_pack", "adamw8_unpack",
    "sharded_stats", "sharded_add_mul_scalar", "sharded_softmax", "sharded_sum_dim",
    "sharded_mean_dim", "sharded_max_dim", "sharded_adamw_update",
]


def version() -> str:
    return lib().rtc_version().decode()


def set_math_mode(mode: str) -> None:
    """"tolerance" (the default: within 1e-6 relative error or 4 ulp of the
    reference's glibc results, single-precision exp/tanh/log) or "exact"
    (glibc's expf/tanhf bit for bit) for the transcendental activations and
    softmax.  Process-wide (rtc_set_math_mode)."""
    code = {"tolerance": _native.MATH_TOLERANCE, "exact": _native.MATH_EXACT}.get(mode)
    if code is None:
        raise ValueError(f"math mode must be 'tolerance' or 'exact', not {mode!r}")
    check(lib().rtc_set_math_mode(code))


def get_math_mode() -> str:
    return "exact" if lib().rtc_get_math_mode() == _native.MATH_EXACT else "tolerance"


class math_mode:
    """Context manager: `with math_mode("exact"): ...` restores the previous
    mode on exit."""

    def __init__(self, mode: str):
        self.mode = mode

    def __enter__(self):
        self.before = get_math_mode()
        set_math_mode(self.mode)
        return self

    def __exit__(self, *exc):
        set_math_mode(self.before)


def synchronize() -> None:
    check(lib().rtc_synchronize())


def _dtype_code(dtype: str) -> int:
    code = _native.DTYPE_NAMES.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be one of {', '.join(_native.DTYPE_NAMES)}, not {dtype!r}")
    return code


# numpy arrays that Tensor.from_numpy takes, beside float32
_INDEX_ARRAYS = {np.dtype(np.int32): "int32", np.dtype(np.int64): "int64",
                 np.dtype(np.float16): "float16"}


class Tensor:
    """A C-contiguous tensor in the memory of one GPU: float32, or for the
    token operators another `dtype` ("bfloat16", "float16", "float8_e4m3",
    "int32", "int64")."""

    def __init__(self, shape, device: int = 0, *, ptr: int | None = None, owner=None,
                 dtype: str = "float32"):
        self._shape = tuple(int(d) for d in shape)
        self.device = int(device)
        self.dtype = dtype
        self._code = _dtype_code(dtype)
        self._owned = ptr is None
        self._owner = owner          # keeps a borrowed buffer alive
        if ptr is None:
            out = c_void_p()
            check(lib().rtc_malloc(self.device, self.nbytes, ctypes.byref(out)))
            ptr = out.value or 0
        self.ptr = int(ptr)
        self._desc = _native.Desc(self.ptr, self._shape, self._code, self.device)

    # ---- construction (rusttorch-py/src/lib.rs:35-61) ---------------------
    @staticmethod
    def zeros(shape, device: int = 0) -> "Tensor":
        return Tensor.from_numpy(np.zeros(list(shape), dtype=np.float32), device)

    @staticmethod
    def ones(shape, device: int = 0) -> "Tensor":
        return Tensor.from_numpy(np.ones(list(shape), dtype=np.float32), device)

    @staticmethod
    def empty(shape, device: int = 0, dtype: str = "float32") -> "Tensor":
        return Tensor(shape, device, dtype=dtype)

    @staticmethod
    def from_numpy(array, device: int = 0, dtype: str | None = None) -> "Tensor":
        """A copy of the array on the GPU: float32, float16, int32 or int64.
        With dtype="bfloat16" float32 values are rounded to it (to nearest,
        ties to even); with dtype="float8_e4m3" uint8 codes are taken as they are."""
        a = np.asarray(array)
        if dtype == "bfloat16" and a.dtype == np.float32:
            a = _bf16_bits(a)
        elif dtype == "float8_e4m3" and a.dtype == np.uint8:
            pass
        else:
            kind = "float32" if a.dtype == np.float32 else _INDEX_ARRAYS.get(a.dtype)
            if kind is None:
                raise RusttorchError("only float32 arrays are supported (float16, int32 and int64 "
                                     "for the token operators)", _native.UNSUPPORTED)
            if dtype not in (None, kind):
                raise RusttorchError(f"a {a.dtype} array does not make a {dtype} tensor",
                                     _native.DTYPE_MISMATCH)
            dtype = kind
        if not a.flags.c_contiguous:
            raise ValueError("Array must be contiguous")
        t = Tensor(a.shape, device, dtype=dtype)
        if t.nbytes:
            check(lib().rtc_memcpy_h2d(t.device, c_void_p(t.ptr), a.ctypes.data_as(c_void_p),
                                       t.nbytes))
        return t

    @staticmethod
    def from_device_ptr(ptr: int, shape, device: int = 0, owner=None,
                        dtype: str = "float32") -> "Tensor":
        """Borrow an existing device buffer (e.g. a torch tensor's data_ptr())."""
        return Tensor(shape, device, ptr=ptr, owner=owner, dtype=dtype)

    # ---- metadata (rusttorch-py/src/lib.rs:63-79) -------------------------
    def shape(self) -> list[int]:
        return list(self._shape)

    def ndim(self) -> int:
        return len(self._shape)

    def numel(self) -> int:
        n = 1
        for d in self._shape:
            n *= d
        return n

    @property
    def nbytes(self) -> int:
        return self.numel() * _native.DTYPE_BYTES[self._code]

    def __repr__(self) -> str:
        return f"Tensor(shape={list(self._shape)}, dtype={self.dtype})"

    def to_numpy(self) -> np.ndarray:
        """The values: bfloat16 as float32, float8_e4m3 as its uint8 codes."""
        out = np.empty(self._shape, dtype={"bfloat16": np.uint16, "float8_e4m3": np.uint8}.get(
            self.dtype, self.dtype))
        if self.nbytes:
            check(lib().rtc_memcpy_d2h(self.device, out.ctypes.data_as(c_void_p),
                                       c_void_p(self.ptr), self.nbytes))
        if self.dtype == "bfloat16":
            return (out.astype(np.uint32) << 16).view(np.float32)
        return out

    @property
    def desc(self):
        """A by-reference rtc_tensor for a C-ABI call.  It holds this tensor
        (and so its device buffer) alive for as long as the reference itself
        is alive, so `Tensor.from_numpy(a).desc` passed straight to a call is
        safe: the temporary tensor is not freed before the call returns."""
        s = _native.RtcTensor.from_buffer_copy(self._desc.s)
        s._owner = self       # the copy -> the tensor; nothing points back
        return ctypes.byref(s)

    def __del__(self):
        try:
            if self._owned and self.ptr:
                lib().rtc_free(self.device, c_void_p(self.ptr))
                self.ptr = 0
        except Exception:
            pass


def _bf16_bits(a: np.ndarray) -> np.ndarray:
    b = np.ascontiguousarray(a).view(np.uint32)
    r = ((b + np.uint32(0x7fff) + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7fc0), r).reshape(a.shape)


class TensorList:
    """Tensors that are passed to a call together, their descriptors laid out
    once: an optimizer keeps one for its parameters, gradients and moments.
    Wherever a function takes a list of tensors it takes one of these.  To lay one
    out takes 0.3 us a tensor, and a Tensor around a pointer 4 us: a program whose
    gradients are other buffers in each step pays both in each."""

    def __init__(self, tensors):
        self.tensors = tuple(tensors)
        self._array = _desc_array(self.tensors)

    def __len__(self) -> int:
        return len(self.tensors)

    def __iter__(self):
        return iter(self.tensors)

    def __getitem__(self, i):
        return self.tensors[i]


def _like(x: Tensor, shape=None) -> Tensor:
    return Tensor(x.shape() if shape is None else shape, x.device)


def _binary(fn, a: Tensor, b: Tensor) -> Tensor:
    out = _like(a)
    check(fn(a.desc, b.desc, out.desc))
    return out


def _unary(fn, x: Tensor, *extra) -> Tensor:
    out = _like(x)
    check(fn(x.desc, out.desc, *extra))
    return out


# ---- elementwise (rusttorch-py/src/lib.rs:83-123, :400-435) ----------------
def add(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_add, a, b)
def mul(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_mul, a, b)
def sub(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_sub, a, b)
def div(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_div, a, b)
def add_simd(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_add_simd, a, b)
def mul_simd(a: Tensor, b: Tensor) -> Tensor: return _binary(lib().rtc_mul_simd, a, b)


def add_scalar(t: Tensor, scalar: float) -> Tensor:
    out = _like(t)
    check(lib().rtc_add_scalar(t.desc, float(scalar), out.desc))
    return out


def mul_scalar(t: Tensor, scalar: float) -> Tensor:
    out = _like(t)
    check(lib().rtc_mul_scalar(t.desc, float(scalar), out.desc))
    return out


def mul_scalar_simd(t: Tensor, scalar: float) -> Tensor:
    out = _like(t)
    check(lib().rtc_mul_scalar_simd(t.desc, float(scalar), out.desc))
    return out


def add_mul_scalar(a: Tensor, b: Tensor, scalar: float) -> Tensor:
    """mul_scalar(add(a, b), scalar) in one pass over memory."""
    out = _like(a)
    check(lib().rtc_add_mul_scalar(a.desc, b.desc, float(scalar), out.desc))
    return out


def fused_multiply_add(a: Tensor, b: Tensor, c: Tensor) -> Tensor:
    out = _like(a)
    check(lib().rtc_fused_multiply_add(a.desc, b.desc, c.desc, out.desc))
    return out


# ---- activations (rusttorch-py/src/lib.rs:126-208) --------------------------
def relu(t: Tensor) -> Tensor: return _unary(lib().rtc_relu, t)
def relu_simd(t: Tensor) -> Tensor: return _unary(lib().rtc_relu_simd, t)
def sigmoid(t: Tensor) -> Tensor: return _unary(lib().rtc_sigmoid, t)
def tanh(t: Tensor) -> Tensor: return _unary(lib().rtc_tanh, t)
def gelu(t: Tensor) -> Tensor: return _unary(lib().rtc_gelu, t)
def swish(t: Tensor) -> Tensor: return _unary(lib().rtc_swish, t)
def selu(t: Tensor) -> Tensor: return _unary(lib().rtc_selu, t)
def mish(t: Tensor) -> Tensor: return _unary(lib().rtc_mish, t)
def softplus(t: Tensor) -> Tensor: return _unary(lib().rtc_softplus, t)
def softsign(t: Tensor) -> Tensor: return _unary(lib().rtc_softsign, t)
def leaky_relu(t: Tensor, alpha: float) -> Tensor: return _unary(lib().rtc_leaky_relu, t, float(alpha))
def elu(t: Tensor, alpha: float) -> Tensor: return _unary(lib().rtc_elu, t, float(alpha))


def softmax(t: Tensor, dim: int) -> Tensor:
    out = _like(t)
    check(lib().rtc_softmax(t.desc, int(dim), out.desc))
    return out


# ---- reductions (rusttorch-py/src/lib.rs:234-242; core reduction.rs) -------
def _scalar(fn, t: Tensor) -> float:
    v = c_double()
    check(fn(t.desc, ctypes.byref(v)))
    return v.value


def sum(t: Tensor) -> float: return _scalar(lib().rtc_sum, t)     # noqa: A001
def mean(t: Tensor) -> float: return _scalar(lib().rtc_mean, t)
def max(t: Tensor) -> float: return _scalar(lib().rtc_max, t)     # noqa: A001
def min(t: Tensor) -> float: return _scalar(lib().rtc_min, t)     # noqa: A001


def stats(t: Tensor) -> tuple[float, float, float, float]:
    """(sum, mean, max, min) from one pass."""
    v = (c_double * 4)()
    check(lib().rtc_stats(t.desc, v))
    return tuple(v)


def _dim(fn, t: Tensor, dim: int) -> Tensor:
    dim = int(dim)
    shape = [d for i, d in enumerate(t.shape()) if i != dim] if 0 <= dim < t.ndim() else []
    out = _like(t, shape)
    check(fn(t.desc, dim, out.desc))
    return out


def sum_dim(t: Tensor, dim: int) -> Tensor: return _dim(lib().rtc_sum_dim, t, dim)
def mean_dim(t: Tensor, dim: int) -> Tensor: return _dim(lib().rtc_mean_dim, t, dim)
def max_dim(t: Tensor, dim: int) -> Tensor: return _dim(lib().rtc_max_dim, t, dim)


# ---- optimizers (rusttorch-py/src/lib.rs:278-369) --------------------------
def adam_update(params, gradients, m, v, learning_rate, beta1, beta2, epsilon, timestep):
    po, mo, vo = _like(params), _like(params), _like(params)
    check(lib().rtc_adam_update(params.desc, gradients.desc, m.desc, v.desc, float(learning_rate),
                                float(beta1), float(beta2), float(epsilon), int(timestep),
                                po.desc, mo.desc, vo.desc))
    return po, mo, vo


def adamw_update(params, gradients, m, v, learning_rate, beta1, beta2, epsilon, weight_decay,
                 timestep):
    po, mo, vo = _like(params), _like(params), _like(params)
    check(lib().rtc_adamw_update(params.desc, gradients.desc, m.desc, v.desc,
                                 float(learning_rate), float(beta1), float(beta2), float(epsilon),
                                 float(weight_decay), int(timestep), po.desc, mo.desc, vo.desc))
    return po, mo, vo


def sgd_update(params, gradients, learning_rate):
    po = _like(params)
    check(lib().rtc_sgd_update(params.desc, gradients.desc, float(learning_rate), po.desc))
    return po


def sgd_momentum_update(params, gradients, velocity, learning_rate, momentum):
    po, vo = _like(params), _like(params)
    check(lib().rtc_sgd_momentum_update(params.desc, gradients.desc, velocity.desc,
                                        float(learning_rate), float(momentum), po.desc, vo.desc))
    return po, vo


# ---- broadcasting (rusttorch-py/src/lib.rs:372-398; core ops/broadcast.rs) ----
def _bshape(a: Tensor, b: Tensor):
    try:
        return list(np.broadcast_shapes(tuple(a.shape()), tuple(b.shape())))
    except ValueError:
        return a.shape()          # the library reports the BroadcastError


def _bcast(fn, a: Tensor, b: Tensor) -> Tensor:
    out = _like(a, _bshape(a, b))
    check(fn(a.desc, b.desc, out.desc))
    return out


def add_broadcast(a: Tensor, b: Tensor) -> Tensor: return _bcast(lib().rtc_add_broadcast, a, b)
def sub_broadcast(a: Tensor, b: Tensor) -> Tensor: return _bcast(lib().rtc_sub_broadcast, a, b)
def mul_broadcast(a: Tensor, b: Tensor) -> Tensor: return _bcast(lib().rtc_mul_broadcast, a, b)
def div_broadcast(a: Tensor, b: Tensor) -> Tensor: return _bcast(lib().rtc_div_broadcast, a, b)


# ---- nn optimizers (core nn/optim.rs), one parameter per call ---------------
def nn_adam_step(params, grads, m, v, lr, beta1, beta2, eps, t):
    """nn::Adam::step for one parameter; t counts steps from 1."""
    po, mo, vo = _like(params), _like(params), _like(params)
    check(lib().rtc_nn_adam_step(params.desc, grads.desc, m.desc, v.desc, float(lr),
                                 float(beta1), float(beta2), float(eps), int(t), po.desc,
                                 mo.desc, vo.desc))
    return po, mo, vo


def nn_sgd_step(params, grads, velocity, lr, momentum=0.0, weight_decay=0.0):
    """nn::SGD::step for one parameter; returns (params', velocity')
    (velocity' is None without momentum)."""
    po = _like(params)
    if momentum > 0.0:
        vo = _like(params)
        check(lib().rtc_nn_sgd_step(params.desc, grads.desc, velocity.desc, float(lr),
                                    float(momentum), float(weight_decay), po.desc, vo.desc))
        return po, vo
    check(lib().rtc_nn_sgd_step(params.desc, grads.desc, None, float(lr), float(momentum),
                                float(weight_decay), po.desc, None))
    return po, None


# ---- autograd backward (core autograd/ops.rs GradFn::backward) -------------
# Each returns what the reference's backward returns for that input; pass
# need_a / need_b False where the reference's operand does not require grad
# (its `None`).
def relu_backward(grad_output: Tensor, input: Tensor) -> Tensor:
    out = _like(grad_output)
    check(lib().rtc_relu_backward(grad_output.desc, input.desc, out.desc))
    return out


def sigmoid_backward(grad_output: Tensor, output: Tensor) -> Tensor:
    out = _like(grad_output)
    check(lib().rtc_sigmoid_backward(grad_output.desc, output.desc, out.desc))
    return out


def tanh_backward(grad_output: Tensor, output: Tensor) -> Tensor:
    out = _like(grad_output)
    check(lib().rtc_tanh_backward(grad_output.desc, output.desc, out.desc))
    return out


def gelu_backward(grad_output: Tensor, input: Tensor) -> Tensor:
    out = _like(input)
    check(lib().rtc_gelu_backward(grad_output.desc, input.desc, out.desc))
    return out


def autograd_gelu(x: Tensor) -> Tensor:
    """autograd's own GELU forward (it rounds differently from gelu)."""
    out = _like(x)
    check(lib().rtc_autograd_gelu(x.desc, out.desc))
    return out


def _pair_out(g: Tensor, need_a: bool, need_b: bool):
    return (_like(g) if need_a else None), (_like(g) if need_b else None)


def _d(t):
    return t.desc if t is not None else None


def add_backward(grad_output: Tensor, need_a=True, need_b=True):
    ga, gb = _pair_out(grad_output, need_a, need_b)
    check(lib().rtc_add_backward(grad_output.desc, _d(ga), _d(gb)))
    return ga, gb


def sub_backward(grad_output: Tensor, need_a=True, need_b=True):
    ga, gb = _pair_out(grad_output, need_a, need_b)
    check(lib().rtc_sub_backward(grad_output.desc, _d(ga), _d(gb)))
    return ga, gb


def mul_backward(grad_output: Tensor, a: Tensor, b: Tensor, need_a=True, need_b=True):
    ga, gb = _pair_out(grad_output, need_a, need_b)
    check(lib().rtc_mul_backward(grad_output.desc, a.desc, b.desc, _d(ga), _d(gb)))
    return ga, gb


def div_backward(grad_output: Tensor, a: Tensor, b: Tensor, need_a=True, need_b=True):
    ga, gb = _pair_out(grad_output, need_a, need_b)
    check(lib().rtc_div_backward(grad_output.desc, a.desc, b.desc, _d(ga), _d(gb)))
    return ga, gb


def sum_backward(grad_output: Tensor, input_shape) -> Tensor:
    out = Tensor(list(input_shape), device=grad_output.device)
    check(lib().rtc_sum_backward(grad_output.desc, out.desc))
    return out


def mean_backward(grad_output: Tensor, input_shape) -> Tensor:
    out = Tensor(list(input_shape), device=grad_output.device)
    check(lib().rtc_mean_backward(grad_output.desc, out.desc))
    return out


def broadcast_add_backward(grad_output: Tensor, a_shape, b_shape, need_a=True, need_b=True):
    ga = Tensor(list(a_shape), device=grad_output.device) if need_a else None
    gb = Tensor(list(b_shape), device=grad_output.device) if need_b else None
    check(lib().rtc_broadcast_add_backward(grad_output.desc, _d(ga), _d(gb)))
    return ga, gb


# ---- loss functions (core ops/loss.rs): Python floats, like rusttorch's f64 --
def _loss(fn, predictions: Tensor, targets: Tensor, *args) -> float:
    v = ctypes.c_double()
    check(fn(predictions.desc, targets.desc, *args, ctypes.byref(v)))
    return v.value


def mse_loss(predictions: Tensor, targets: Tensor) -> float:
    return _loss(lib().rtc_mse_loss, predictions, targets)


def l1_loss(predictions: Tensor, targets: Tensor) -> float:
    return _loss(lib().rtc_l1_loss, predictions, targets)


def smooth_l1_loss(predictions: Tensor, targets: Tensor, beta: float = 1.0) -> float:
    return _loss(lib().rtc_smooth_l1_loss, predictions, targets, float(beta))


def binary_cross_entropy_loss(predictions: Tensor, targets: Tensor, epsilon: float = 1e-7) -> float:
    return _loss(lib().rtc_binary_cross_entropy_loss, predictions, targets, float(epsilon))


def cross_entropy_loss(predictions: Tensor, targets: Tensor, epsilon: float = 1e-7) -> float:
    return _loss(lib().rtc_cross_entropy_loss, predictions, targets, float(epsilon))


# ---- token operators ---------------------------------------------------------
# Asynchronous; with `out`, `loss`, `stats` and `grad` given (buffers that a
# training loop keeps) a call allocates nothing from Python.  The descriptors go
# in as they are (_desc.ref): the arguments live until the call returns.
def embedding(weight: Tensor, ids: Tensor, scale: float = 1.0, out: Tensor | None = None) -> Tensor:
    """weight[ids] * scale: weight [V, D] in float32, bfloat16 or float16, ids
    of any shape in int32 or int64."""
    if out is None:
        width = weight.shape()[1:] if weight.ndim() == 2 else []
        out = Tensor(ids.shape() + width, weight.device, dtype=weight.dtype)
    check(lib().rtc_embedding(weight._desc.ref, ids._desc.ref, float(scale), out._desc.ref))
    return out


def embedding_backward(grad_output: Tensor, ids: Tensor, num_embeddings: int, scale: float = 1.0,
                       padding_idx: int | None = None, accumulate: bool = False,
                       out: Tensor | None = None) -> Tensor:
    """The gradient of embedding()'s weight, [num_embeddings, D], in float32
    unless `out` has grad_output's type.  With accumulate, it is added to
    `out`, of which only the rows that ids name are touched."""
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        width = grad_output.shape()[-1:]
        out = Tensor([int(num_embeddings)] + width, grad_output.device)
    elif out.ndim() == 2 and out.shape()[0] != num_embeddings:
        raise RusttorchError(f"out has {out.shape()[0]} rows, num_embeddings is {num_embeddings}",
                             _native.SHAPE_MISMATCH)
    padding = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and padding < 0:
        raise RusttorchError("padding_idx must not be negative", _native.INVALID_ARGUMENT)
    check(lib().rtc_embedding_backward(grad_output._desc.ref, ids._desc.ref, float(scale), padding,
                                       int(accumulate), out._desc.ref))
    return out


def _reduction(reduction: str) -> int:
    code = _native.REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', not {reduction!r}")
    return code


def _loss_out(targets: Tensor, reduction: str, loss: Tensor | None) -> Tensor:
    if loss is not None:
        return loss
    return Tensor(targets.shape() if reduction == "none" else [], targets.device)


def softmax_cross_entropy(logits: Tensor, targets: Tensor, ignore_index: int = -100,
                          reduction: str = "mean", loss: Tensor | None = None,
                          stats: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(loss, stats) of logits [..., V] against token ids: loss a float32
    tensor on the GPU, stats what softmax_cross_entropy_backward needs."""
    code = _reduction(reduction)
    loss = _loss_out(targets, reduction, loss)
    if stats is None:
        stats = Tensor(targets.shape() + [3], targets.device)
    check(lib().rtc_softmax_cross_entropy(logits._desc.ref, targets._desc.ref, int(ignore_index),
                                          code, loss._desc.ref, stats._desc.ref))
    return loss, stats


def softmax_cross_entropy_backward(grad_output: Tensor, logits: Tensor, targets: Tensor,
                                   stats: Tensor, ignore_index: int = -100,
                                   reduction: str = "mean", out: Tensor | None = None) -> Tensor:
    """The gradient of softmax_cross_entropy's logits (out may be logits)."""
    code = _reduction(reduction)
    if out is None:
        out = Tensor(logits.shape(), logits.device, dtype=logits.dtype)
    check(lib().rtc_softmax_cross_entropy_backward(
        grad_output._desc.ref, logits._desc.ref, targets._desc.ref, stats._desc.ref,
        int(ignore_index), code, out._desc.ref))
    return out


def softmax_cross_entropy_grad(logits: Tensor, targets: Tensor, ignore_index: int = -100,
                               reduction: str = "mean", grad_scale: float = 1.0,
                               loss: Tensor | None = None,
                               grad: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(loss, gradient of the logits times grad_scale) in one pass where a row
    fits on chip (grad may be logits)."""
    code = _reduction(reduction)
    loss = _loss_out(targets, reduction, loss)
    if grad is None:
        grad = Tensor(logits.shape(), logits.device, dtype=logits.dtype)
    check(lib().rtc_softmax_cross_entropy_grad(logits._desc.ref, targets._desc.ref,
                                               int(ignore_index), code, float(grad_scale),
                                               loss._desc.ref, grad._desc.ref))
    return loss, grad


def adamw_update_multi(params, grads, m, v, learning_rate, beta1, beta2, epsilon, weight_decay,
                       timestep, m_scales=None, v_scales=None, copies=None, seed: int = 0) -> None:
    """adamw_update of many tensors in place, in few launches (lists of
    Tensors, or TensorLists).  grads may be float32, bfloat16 or float16.  With
    float8_e4m3 m and v and their scales (adamw8_pack) the moments are held in
    8 bits, rounded stochastically from `seed` (another one each step).  copies
    (bfloat16 or float16) receive the rounded parameters."""
    lists = [params, grads, m, v, m_scales, v_scales, copies]
    lists = [t if t is None or isinstance(t, TensorList) else TensorList(t) for t in lists]
    n = len(lists[0])
    if any(t is not None and len(t) != n for t in lists):
        raise ValueError("every list must have as many tensors as params")
    check(lib().rtc_adamw_update_multi(*(t._array if t is not None else None for t in lists), n,
                                       learning_rate, beta1, beta2, epsilon, weight_decay,
                                       int(timestep), int(seed)))


def adamw8_pack(m: Tensor, v: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(m_codes, m_scales, v_codes, v_scales) of float32 moments, to nearest."""
    blocks = [-(-m.numel() // _native.MOMENT_BLOCK)]
    mc, vc = (Tensor(m.shape(), m.device, dtype="float8_e4m3") for _ in range(2))
    ms, vs = Tensor(blocks, m.device), Tensor(blocks, m.device)
    check(lib().rtc_adamw8_pack(m._desc.ref, v._desc.ref, mc._desc.ref, ms._desc.ref, vc._desc.ref,
                                vs._desc.ref))
    return mc, ms, vc, vs


def adamw8_unpack(m_codes: Tensor, m_scales: Tensor, v_codes: Tensor,
                  v_scales: Tensor) -> tuple[Tensor, Tensor]:
    """The float32 moments that adamw8_pack's or a step's codes stand for."""
    m, v = _like(m_codes), _like(m_codes)
    check(lib().rtc_adamw8_unpack(m_codes._desc.ref, m_scales._desc.ref, v_codes._desc.ref,
                                  v_scales._desc.ref, m._desc.ref, v._desc.ref))
    return m, v


# ---- one process, several GPUs ---------------------------------------------
def sharded_stats(shards) -> tuple[float, float, float, float]:
    """(sum, mean, max, min) of the concatenation of `shards` (Tensors, each
    on its own GPU or not), every shard summarised on its device at once."""
    shards = list(shards)
    arr = (_native.RtcTensor * (len(shards) or 1))()
    for i, t in enumerate(shards):
        arr[i] = t._desc.s
    out = (c_double * 4)()
    check(lib().rtc_sharded_stats(arr, len(shards), out))
    return out[0], out[1], out[2], out[3]


def _desc_array(tensors):
    arr = (_native.RtcTensor * (len(tensors) or 1))()
    for i, t in enumerate(tensors):
        arr[i] = t._desc.s
    return arr


def _like_shards(shards, shapes=None):
    return [_like(t, shapes[i] if shapes else None) for i, t in enumerate(shards)]


def sharded_add_mul_scalar(a, b, scalar: float):
    """mul_scalar(add(a, b), scalar) of a tensor split into shards (lists of
    Tensors, shard i of a and b on one GPU): one new Tensor per shard."""
    a, b = list(a), list(b)
    if len(a) != len(b):
        raise ValueError("a and b must have the same number of shards")
    out = _like_shards(a)
    check(lib().rtc_sharded_add_mul_scalar(_desc_array(a), _desc_array(b), float(scalar),
                                           _desc_array(out), len(a)))
    return out


def sharded_softmax(shards, dim: int):
    """softmax along `dim` of row blocks (the shards split axis 0)."""
    shards = list(shards)
    out = _like_shards(shards)
    check(lib().rtc_sharded_softmax(_desc_array(shards), dim, _desc_array(out), len(shards)))
    return out


def _sharded_dim(fn, shards, dim: int):
    shards = list(shards)
    dim = int(dim)
    out = _like_shards(shards, [[d for k, d in enumerate(t.shape()) if k != dim]
                                if 0 <= dim < t.ndim() else [] for t in shards])
    check(fn(_desc_array(shards), dim, _desc_array(out), len(shards)))
    return out


def sharded_sum_dim(shards, dim: int):
    """sum_dim of each shard on its own GPU (the shards split an axis other
    than dim: column blocks for dim 0, row blocks for the last axis)."""
    return _sharded_dim(lib().rtc_sharded_sum_dim, shards, dim)


def sharded_mean_dim(shards, dim: int):
    return _sharded_dim(lib().rtc_sharded_mean_dim, shards, dim)


def sharded_max_dim(shards, dim: int):
    return _sharded_dim(lib().rtc_sharded_max_dim, shards, dim)


def sharded_adamw_update(params, grads, m, v, learning_rate, beta1, beta2, epsilon, weight_decay,
                         timestep):
    """adamw_update of every shard, in place (params, m, v are updated)."""
    params, grads, m, v = list(params), list(grads), list(m), list(v)
    if not len(params) == len(grads) == len(m) == len(v):
        raise ValueError("params, grads, m and v must have the same number of shards")
    check(lib().rtc_sharded_adamw_update(_desc_array(params), _desc_array(grads), _desc_array(m),
                                         _desc_array(v), learning_rate, beta1, beta2, epsilon,
                                         weight_decay, int(timestep), len(params)))
