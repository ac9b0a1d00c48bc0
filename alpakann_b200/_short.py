"""The short way to the decode operators on compressed data.

`binding` is the compiled module of binding/binding.c (a call costs 4 us of host time), or,
where it cannot be had -- not built, built for another interpreter, a torch without
DLPack's C exchange interface -- an object with the same functions through ctypes
(25 us). Each takes the stream handle (None: the current stream), the tensors (None
where optional) and the scalars in the order of the C call, and returns the C
call's code, or MISMATCH or ELSEWHERE when nothing was called.
"""
import ctypes
import importlib.util
import os
import sysconfig

import torch

from ._capi import HERE, MAX_RANK, SIGNATURES, lib, ref

MISMATCH, ELSEWHERE = -1, -3  # unfit tensors, or on a device that is not the current one
PATH = os.path.join(HERE, "_build", "_ann_binding" + sysconfig.get_config_var("EXT_SUFFIX"))


def _compiled():
    """The compiled module, or None."""
    if not os.path.exists(PATH):
        return None
    spec = importlib.util.spec_from_file_location("_ann_binding", PATH)
    try:
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.setup(torch.Tensor, torch._C._cuda_getDevice)
    except (ImportError, AttributeError, ValueError):
        return None
    return module


class ThroughCtypes:
    """The compiled module's functions, slower."""


def _entry(c_name, types, optional):
    fn, scalars = getattr(lib, c_name), SIGNATURES[c_name][0][1 + len(types):]
    limits = {ctypes.c_uint32: (0, 2**32 - 1), ctypes.c_int32: (-2**31, 2**31 - 1)}

    def whole(kind, value):
        if kind not in limits:
            return float(value)
        low, high = limits[kind]
        value = int(value)
        if not low <= value <= high:
            raise OverflowError("integer argument out of range")
        return value

    def call(stream, *args):
        if len(args) != len(types) + len(scalars):
            raise TypeError("wrong number of arguments")
        device, views = None, []
        for i, (t, want) in enumerate(zip(args, types)):
            if t is None and i in optional:
                views.append(None)
                continue
            fits = isinstance(t, torch.Tensor) and t.is_cuda and t.dim() <= MAX_RANK and (
                t.dtype == want or (want == torch.int32 and t.dtype == torch.uint32))
            if not fits or (device is not None and t.device != device):
                return MISMATCH
            device = t.device
            views.append(ref(t))
        if device.index != torch.cuda.current_device():
            return ELSEWHERE
        values = [whole(kind, v) for kind, v in zip(scalars, args[len(types):])]
        if stream is None:
            stream = torch.cuda.current_stream(device).cuda_stream
        return fn(stream, *views, *values)

    return call


def _through_ctypes():
    f32, f64, i8, i32 = torch.float32, torch.float64, torch.int8, torch.int32
    binding = ThroughCtypes()
    for name, t in (("rotary_f32", f32), ("rotary_f64", f64)):
        setattr(binding, name, _entry(f"ann_{name}", [t, t, i32, f64, t, t], (1, 5)))
    binding.kv_cache_append_q8 = _entry("ann_kv_cache_append_q8_f32", [f32, f32, i8, i8, f32, f32, i32, i32], (7,))
    binding.kv_cache_read_q8 = _entry("ann_kv_cache_read_q8_f32", [i8, i8, f32, f32, f32, f32, i32], (6,))
    binding.attention_decode_q8 = _entry("ann_attention_decode_q8_f32", [f32, i8, i8, f32, f32, i32, f32], (5,))
    binding.linear_q4 = _entry("ann_linear_q4_f32", [f32, i32, f32, f32, f32, f32], (3, 4))
    return binding


binding = _compiled() or _through_ctypes()
