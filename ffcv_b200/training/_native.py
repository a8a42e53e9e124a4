"""Calls of ``libffcv_b200.so`` for the training step: arguments are packed into the C structures of
``include/ffcv_b200.h`` (all 8-byte members first, so that there is no padding)."""
import struct
from ctypes import c_char_p, c_int, c_int32, c_int64, c_void_p

import torch as ch
from torch._C._dynamo.guards import TensorGuards

from ..libffcv import lib

TYPES = {ch.float32: 0, ch.float16: 1, ch.bfloat16: 2}

CROSS_ENTROPY = struct.Struct('=8Q6q8i2f')
LINEAR_CROSS_ENTROPY = struct.Struct('=11Q7q8i2f')
DISTILLATION = struct.Struct('=10Q9q10i4f')
DISTILLATION_MOST = 1024
GROUP_NORM = struct.Struct('=9Q8q4ifi')
NORM_RESIDUAL = struct.Struct('=21Q8q6i2f')
ROTARY = struct.Struct('=7Q19q6ifi')
ADAMW = struct.Struct('=7Qq4id')
ADAMW_GROUP = struct.Struct('=5d')
ADAMW_BLOCK = 256
NORM_MAX_WIDTH = 16384

lib.ffcvb_training_error.argtypes = []
lib.ffcvb_training_error.restype = c_char_p
for _name in ('ffcvb_cross_entropy', 'ffcvb_distillation', 'ffcvb_norm_residual', 'ffcvb_norm_residual_backward', 'ffcvb_rotary'):
    getattr(lib, _name).argtypes = [c_char_p, c_void_p]
    getattr(lib, _name).restype = c_int
lib.ffcvb_norm_residual_backward.argtypes = [c_char_p, c_void_p, c_void_p]
lib.ffcvb_norm_residual_workspace.argtypes = [c_char_p]
lib.ffcvb_norm_residual_workspace.restype = c_int64
lib.ffcvb_group_norm.argtypes = lib.ffcvb_group_norm_backward.argtypes = [c_char_p, c_void_p, c_void_p]
lib.ffcvb_group_norm.restype = lib.ffcvb_group_norm_backward.restype = c_int
lib.ffcvb_group_norm_workspace.argtypes = [c_char_p, c_int]
lib.ffcvb_group_norm_workspace.restype = c_int64
lib.ffcvb_linear_cross_entropy.argtypes = [c_char_p, c_void_p, c_void_p]
lib.ffcvb_linear_cross_entropy.restype = c_int
lib.ffcvb_linear_cross_entropy_workspace.argtypes = [c_char_p]
lib.ffcvb_linear_cross_entropy_workspace.restype = c_int64
lib.ffcvb_adamw_layout.argtypes = [c_int32, c_void_p, c_void_p, c_void_p]
lib.ffcvb_adamw_layout.restype = c_int64
lib.ffcvb_adamw_table.argtypes = [c_int32, c_void_p, c_void_p, c_void_p]
lib.ffcvb_adamw_table.restype = c_int
lib.ffcvb_adamw_step.argtypes = [c_char_p, c_void_p, c_void_p, c_void_p, c_char_p, c_char_p, c_int32, c_void_p]
lib.ffcvb_adamw_step.restype = c_int
lib.ffcvb_adamw_masters.argtypes = [c_char_p, c_void_p, c_char_p, c_void_p]
lib.ffcvb_adamw_masters.restype = c_int


def check(rc):
    if rc != 0:
        raise RuntimeError(f'{lib.ffcvb_training_error().decode()} (error {rc})')


# The handle of a device's current stream, without the object around it that ch.cuda.current_stream makes (2 us a call).
raw_stream = ch._C._cuda_getCurrentRawStream
# Whether the current stream of the current device is being captured in a graph.
capturing = ch._C._cuda_isCurrentStreamCapturing


def layouts(tensors):
    """What tensors are, whatever their values: ``layouts(a).check(*b)`` says whether sizes, strides, types and devices of b are those of a, of
    148 tensors in 15 us (their strides, sizes and types as Python sees them take 40)."""
    return TensorGuards(*tensors, dynamic_dims_sizes=None, dynamic_dims_strides=None)


def stream_of(tensor):
    return raw_stream(tensor.get_device())


def ptr(tensor):
    return 0 if tensor is None else tensor.data_ptr()


def new_like(t):
    """Room for a contiguous result of a tensor's shape and type."""
    return ch.empty_like(t) if t.is_contiguous() else ch.empty(t.shape, dtype=t.dtype, device=t.device)


def require(tensor, name, like=None):
    """A CUDA tensor of a type the kernels know, on the device of `like`."""
    if not isinstance(tensor, ch.Tensor):
        raise TypeError(f'{name} is not a tensor')
    if not tensor.is_cuda:
        raise TypeError(f'{name} is not on a GPU; ffcv_b200 has no CPU form of this operator')
    if tensor.dtype not in TYPES:
        raise TypeError(f'{name}: {tensor.dtype} is none of float32, float16, bfloat16')
    if like is not None and tensor.device != like.device:
        raise ValueError(f'{name} is on {tensor.device}, not on {like.device}')
    return TYPES[tensor.dtype]
