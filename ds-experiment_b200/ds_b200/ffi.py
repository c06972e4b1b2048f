"""Custom-call surface of libds_b200, shaped like the reference's jax.ffi use.

The reference registers its XLA-FFI handlers by target name and calls them
with ``ffi.ffi_call(name, ShapeDtypeStruct(...), vmap_method=...)(*args,
**attrs)`` (python/test_ds_add.py:16-48,
python/test_ds_recurrence_add_mul_to_f64_cuda.py:18-31).  This module keeps
that surface over torch CUDA tensors: ``register_ffi_target(name, lib.<sym>,
platform="CUDA")`` binds a target name to a libds_b200 entry point, and
``ffi_call`` allocates the results, passes torch's current CUDA stream and
raises on a non-OK status.  Every reference target name is registered at
import.  Scratch for ds_reduce / ds_dot_general comes from torch's caching
allocator (the role XLA's scratch allocator plays for an FFI handler); small
scratch is kept per stream and host thread and reused, and a reduce's scratch
size is asked once per shape.
"""
from __future__ import annotations

import array
import ctypes
import threading
from dataclasses import dataclass
from typing import Dict, Tuple

import torch

from . import _lib


@dataclass(frozen=True)
class ShapeDtypeStruct:
    shape: Tuple[int, ...]
    dtype: torch.dtype

    def __init__(self, shape, dtype):
        object.__setattr__(self, "shape", tuple(int(d) for d in shape))
        object.__setattr__(self, "dtype", dtype)


F64, F32, S32 = torch.float64, torch.float32, torch.int32


@dataclass(frozen=True)
class _Convention:
    """Operand dtypes, attribute names and result dtypes of one entry point,
    in the order of the reference handler's Bind() (Args, Attrs, Rets)."""
    args: Tuple[torch.dtype, ...]
    attrs: Tuple[str, ...]
    results: Tuple[torch.dtype, ...]
    kind: str = "plain"  # plain | reduce | reduce_f64 | dot | dot_f64 | scan | ragged | ...
    optional: Tuple[int, ...] = ()  # operands that may be None


CONVENTIONS: Dict[str, _Convention] = {
    "ds_from_f64": _Convention((F64,), (), (F32,)),
    "ds_to_f64": _Convention((F32,), (), (F64,)),
    "ds_from_f32": _Convention((F32,), (), (F32,)),
    "ds_to_f32": _Convention((F32,), (), (F32,)),
    "ds_add": _Convention((F32, F32), (), (F32,)),
    "ds_sub": _Convention((F32, F32), (), (F32,)),
    "ds_mul": _Convention((F32, F32), (), (F32,)),
    "ds_fused_add_mul": _Convention((F64, F64), (), (F32,)),
    "ds_fused_add_mul_to_f64": _Convention((F64, F64), (), (F64,)),
    "ds_fused_axpy": _Convention((F64, F64), (), (F64,)),
    "ds_fused_add_mul_to_f64_cuda": _Convention((F64, F64), (), (F64,)),
    "ds_fused_add_sub_to_f64_cuda": _Convention((F64, F64), (), (F64,)),
    "ds_recurrence_add_mul_to_f64_cuda": _Convention((F64, F64), ("k",), (F64,)),
    "ds_fused_add_mul3_to_f64": _Convention((F64, F64, F64), (), (F64,)),
    "ds_recurrence_mul_add_to_f64": _Convention((F64, F64, F64), ("k",), (F64,)),
    "ds_reduce": _Convention((F32, F32, F32, F32), ("dimensions", "body"), (F32, F32),
                             "reduce"),
    "ds_reduce_f64": _Convention((F64, F64), ("dimensions", "body"), (F64,), "reduce_f64"),
    "ds_reduce_from_f64": _Convention((F64, F64), ("dimensions", "body"), (F32, F32),
                                      "reduce_from_f64"),
    "ds_reduce_packed": _Convention((F32, F32, F32), ("dimensions", "body"), (F32, F32),
                                    "reduce_packed"),
    "ds_dot_general": _Convention((F32, F32, F32, F32),
                                  ("lhs_batching_dimensions", "rhs_batching_dimensions",
                                   "lhs_contracting_dimensions",
                                   "rhs_contracting_dimensions", "algorithm"),
                                  (F32, F32), "dot"),
    "ds_dot_general_f64": _Convention((F64, F64),
                                      ("lhs_batching_dimensions", "rhs_batching_dimensions",
                                       "lhs_contracting_dimensions",
                                       "rhs_contracting_dimensions", "algorithm"),
                                      (F64,), "dot_f64"),
    "ds_linear_recurrence_f64": _Convention((F64, F64, F64), (), (F64,), "scan", (2,)),
    "ds_linear_recurrence_f32": _Convention((F32, F32, F32), (), (F32,), "scan", (2,)),
    "ds_linear_recurrence_packed": _Convention((F32, F32, F32), (), (F32,), "scan", (2,)),
    "ds_linear_recurrence_vjp_f64": _Convention((F64,) * 4, (), (F64,) * 3, "scan", (3,)),
    "ds_linear_recurrence_vjp_f32": _Convention((F32,) * 4, (), (F32,) * 3, "scan", (3,)),
    "ds_linear_recurrence_vjp_packed": _Convention((F32,) * 4, (), (F32,) * 3, "scan", (3,)),
    "ds_ragged_dot": _Convention((F32, F32, F32, F32, S32), ("rhs_contracting", "algorithm"),
                                 (F32, F32), "ragged"),
    "ds_ragged_dot_f64": _Convention((F64, F64, S32), ("rhs_contracting", "algorithm"), (F64,),
                                     "ragged"),
    "ds_ragged_dot_contract": _Convention((F32, F32, F32, F32, S32), ("algorithm",), (F32, F32),
                                          "ragged_contract"),
    "ds_ragged_dot_contract_f64": _Convention((F64, F64, S32), ("algorithm",), (F64,),
                                              "ragged_contract"),
}

# The reference's target names, each bound to its replacement entry point.
REFERENCE_TARGETS = {
    "ds_from_f64": "ds_from_f64",
    "ds_to_f64": "ds_to_f64",
    "ds_from_f32": "ds_from_f32",
    "ds_to_f32": "ds_to_f32",
    "ds_add": "ds_add",
    "ds_sub": "ds_sub",
    "ds_mul": "ds_mul",
    "ds_fused_add_mul": "ds_fused_add_mul",
    "ds_fused_add_mul_to_f64": "ds_fused_add_mul_to_f64",
    "ds_fused_axpy": "ds_fused_axpy",
    "ds_fused_add_mul_to_f64_cuda": "ds_fused_add_mul_to_f64_cuda",
    "ds_fused_add_sub_to_f64_cuda": "ds_fused_add_sub_to_f64_cuda",
    "ds_recurrence_add_mul_to_f64_cuda": "ds_recurrence_add_mul_to_f64_cuda",
    "ds_fused_add_mul3_to_f64": "ds_fused_add_mul3_to_f64",
    "ds_recurrence_mul_add_to_f64": "ds_recurrence_mul_add_to_f64",
    "ds_reduce": "ds_reduce",
    "ds_reduce_f64": "ds_reduce_f64",
    "ds_reduce_from_f64": "ds_reduce_from_f64",
    "ds_reduce_packed": "ds_reduce_packed",
    "ds_dot_general": "ds_dot_general",
    "ds_dot_general_f64": "ds_dot_general_f64",
}

# Targets without a counterpart in the reference: the recurrence along a
# sequence and the products grouped by expert, with their gradients.
SEQUENCE_TARGETS = {name: name for name, c in CONVENTIONS.items()
                    if c.kind in ("scan", "ragged", "ragged_contract")}

# target name -> libds_b200 symbol; every target is bound at import.
_registry: Dict[str, str] = {**REFERENCE_TARGETS, **SEQUENCE_TARGETS}


def register_ffi_target(name: str, target, platform: str = "CUDA") -> None:
    """Bind custom-call target `name` to a libds_b200 entry point.

    `target` is a ctypes function of libds_b200 (``lib.ds_add``) or its
    symbol name.  Only platform "CUDA" exists: there is no host fallback.
    """
    if platform.upper() not in ("CUDA", "GPU"):
        raise ValueError(f"platform {platform!r} is not provided; libds_b200 runs on CUDA only")
    sym = target if isinstance(target, str) else getattr(target, "__name__", None)
    if sym not in CONVENTIONS:
        raise ValueError(f"{sym!r} is not a libds_b200 entry point")
    _registry[name] = sym
    _calls.clear()


def registered_targets():
    return sorted(_registry)


def _stream_handle(device=None) -> ctypes.c_void_p:
    return ctypes.c_void_p(_lib.current_stream_ptr(device))


def _check_tensor(t, dtype, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{what}: libds_b200 operates on CUDA tensors only")
    if t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: tensor must be contiguous (row-major)")


def _buf(t):
    return _lib.make_buffer(t.data_ptr(), t.shape)


# Workspaces up to _CACHED_WORKSPACE_MAX (reduce partials, the residue
# planes of products up to about 1100 x 1100) are kept per (device, stream,
# host thread) and reused: one thread's calls on one stream run in order, so one
# buffer serves them all, and a call skips an allocation.  (Two threads that
# launch on one stream take turns launch by launch, and a call has several.)
# They end with their thread.  The buffer starts at 1 MiB and grows
# to the next power of two a request needs; the one it replaces was
# allocated on the same stream, so torch's allocator hands its memory out
# again only to work ordered after the calls that used it.  Larger ones come
# from torch's allocator each time, so that they are not held.  None is kept
# while a CUDA graph is being captured (its replay may overlap eager calls).
_SMALL_WORKSPACE = 1 << 20
_CACHED_WORKSPACE_MAX = 64 << 20
_workspaces: Dict[tuple, torch.Tensor] = {}
_thread = threading.local()


class _ThreadKeys(set):
    """The keys of a thread's workspaces, held by the thread."""

    def __del__(self):
        for key in self if _workspaces is not None else ():  # None: the interpreter ends
            _workspaces.pop(key, None)


def _workspace(nbytes: int, device, stream: int = 0) -> torch.Tensor:
    nbytes = max(int(nbytes), 1)
    if nbytes > _CACHED_WORKSPACE_MAX or torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, stream, threading.get_ident())
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is None and len(_workspaces) > 64:
            _workspaces.clear()
        if not hasattr(_thread, "keys"):
            _thread.keys = _ThreadKeys()
        _thread.keys.add(key)
        size = max(_SMALL_WORKSPACE, 1 << (nbytes - 1).bit_length())
        ws = _workspaces[key] = torch.empty(size, dtype=torch.uint8, device=device)
    return ws


# ds_reduce_workspace_size by (device, shape, dimensions): a pure function
# of them, asked on every reduce call otherwise.  Likewise the dot_general's
# dimension-number struct and ds_dot_general_workspace_size, by (target,
# device, shapes, algorithm, dimension numbers).
_reduce_ws: Dict[tuple, int] = {}
_dot_setup: Dict[tuple, tuple] = {}
_dims_arrays: Dict[tuple, object] = {}


def _dims_array(dims: tuple):
    arr = _dims_arrays.get(dims)
    if arr is None:
        if len(_dims_arrays) > 256:
            _dims_arrays.clear()
        arr = _dims_arrays[dims] = (ctypes.c_int64 * max(len(dims), 1))(*dims)
    return arr


# (target, result specs) -> the callable ffi_call built for them
_calls: Dict[tuple, object] = {}
_MAX_CALLS = 512


def ffi_call(target_name: str, result_shape_dtypes, vmap_method=None):
    """Return a callable running target `target_name` on torch CUDA tensors.

    result_shape_dtypes: a ShapeDtypeStruct or a sequence of them, one per
    result.  Attributes are keyword arguments, as in jax.ffi.ffi_call.
    vmap_method is accepted for signature compatibility; the entry points
    already take arbitrary leading (batch) dimensions.  Callables are cached
    per target and result specs, so a call site that asks again each time
    pays a dictionary lookup.
    """
    key = (target_name, result_shape_dtypes if isinstance(result_shape_dtypes, ShapeDtypeStruct)
           else tuple(result_shape_dtypes))
    hit = _calls.get(key)
    if hit is not None:
        return hit
    call = _make_call(target_name, result_shape_dtypes)
    if len(_calls) >= _MAX_CALLS:
        _calls.clear()
    _calls[key] = call
    return call


def _make_call(target_name: str, result_shape_dtypes):
    if target_name not in _registry:
        raise KeyError(f"custom-call target {target_name!r} is not registered")
    sym = _registry[target_name]
    conv = CONVENTIONS[sym]
    fn = getattr(_lib.lib(), sym)
    single = isinstance(result_shape_dtypes, ShapeDtypeStruct)
    results_spec = [result_shape_dtypes] if single else list(result_shape_dtypes)
    if len(results_spec) != len(conv.results):
        raise ValueError(f"{target_name}: expected {len(conv.results)} result(s)")
    for spec, dt in zip(results_spec, conv.results):
        if spec.dtype != dt:
            raise TypeError(f"{target_name}: result dtype must be {dt}, got {spec.dtype}")

    def call(*args: torch.Tensor, out=None, **attrs):
        """Run the target.  `out`: optional pre-allocated result tensor(s)
        (contiguous, of the declared shapes and dtypes), as XLA hands a
        handler its result buffers; otherwise results are allocated."""
        if len(args) != len(conv.args):
            raise TypeError(f"{target_name}: expected {len(conv.args)} operand(s), got {len(args)}")
        for i, (t, dt) in enumerate(zip(args, conv.args)):
            if t is None and i in conv.optional:
                continue
            _check_tensor(t, dt, f"{target_name} operand {i}")
        unknown = set(attrs) - set(conv.attrs)
        if unknown:
            raise TypeError(f"{target_name}: unknown attribute(s) {sorted(unknown)}")
        device = args[0].device
        if out is not None:
            out = [out] if isinstance(out, torch.Tensor) else list(out)
            if len(out) != len(results_spec):
                raise ValueError(f"{target_name}: expected {len(results_spec)} output tensor(s)")
            for i, (t, s) in enumerate(zip(out, results_spec)):
                _check_tensor(t, s.dtype, f"{target_name} result {i}")
                if tuple(t.shape) != s.shape:
                    raise ValueError(f"{target_name} result {i}: shape {tuple(t.shape)} != {s.shape}")
        if device.index is not None and device.index != torch.cuda.current_device():
            with torch.cuda.device(device):
                return _invoke(args, attrs, device, out)
        return _invoke(args, attrs, device, out)

    def _invoke(args, attrs, device, out):
        if conv.kind in _SEQUENCE_KINDS:
            outs = _invoke_sequence(target_name, sym, conv, results_spec, args, attrs, device, out)
            return outs[0] if single else tuple(outs)
        outs = out if out is not None else [
            torch.empty(s.shape, dtype=s.dtype, device=device) for s in results_spec]
        keep = []
        bufs = []
        for t in list(args) + outs:
            b, d = _buf(t)
            keep.append(d)
            bufs.append(b)
        refs = [ctypes.byref(b) for b in bufs]
        stream_ptr = _lib.current_stream_ptr(device)
        stream = ctypes.c_void_p(stream_ptr)
        if conv.kind == "plain":
            call_args = refs[:len(args)]
            for name in conv.attrs:
                if name not in attrs:
                    raise TypeError(f"{target_name}: missing attribute {name!r}")
                call_args.append(int(attrs[name]))
            call_args += refs[len(args):]
            status = fn(*call_args, stream)
        elif conv.kind in ("reduce", "reduce_f64", "reduce_from_f64", "reduce_packed"):
            dims = tuple(int(d) for d in attrs.get("dimensions", ()))
            body = int(attrs.get("body", _lib.DS_BODY_ADD))
            cdims = _dims_array(dims)
            shape = tuple(args[0].shape[:-1]) if conv.kind == "reduce_packed" else tuple(args[0].shape)
            wkey = (device.index, shape, dims)
            ws_bytes = _reduce_ws.get(wkey)
            if ws_bytes is None:
                if conv.kind == "reduce_packed":  # sized on the logical shape [..., 2] -> [...]
                    lb, ld = _lib.make_buffer(args[0].data_ptr(), shape)
                    keep.append(ld)
                    ws_bytes = _lib.lib().ds_reduce_workspace_size(ctypes.byref(lb), cdims,
                                                                   len(dims))
                else:
                    ws_bytes = _lib.lib().ds_reduce_workspace_size(refs[0], cdims, len(dims))
                if len(_reduce_ws) > 1024:
                    _reduce_ws.clear()
                _reduce_ws[wkey] = ws_bytes
            ws = _workspace(ws_bytes, device, stream_ptr)
            wsp = ctypes.c_void_p(ws.data_ptr())
            if conv.kind == "reduce":
                status = fn(refs[0], refs[1], refs[2], refs[3], cdims, len(dims), body,
                            refs[4], refs[5], wsp, ws_bytes, stream)
            elif conv.kind == "reduce_f64":
                status = fn(refs[0], refs[1], cdims, len(dims), body, refs[2], wsp,
                            ws_bytes, stream)
            elif conv.kind == "reduce_packed":
                status = fn(refs[0], refs[1], refs[2], cdims, len(dims), body, refs[3], refs[4],
                            wsp, ws_bytes, stream)
            else:
                status = fn(refs[0], refs[1], cdims, len(dims), body, refs[2], refs[3],
                            wsp, ws_bytes, stream)
        else:
            algorithm = int(attrs.get("algorithm", _lib.DS_DOT_TENSOR_INT8))
            rhs = args[2] if conv.kind == "dot" else args[1]
            dkey = (conv.kind, device.index, tuple(args[0].shape), tuple(rhs.shape), algorithm,
                    tuple(attrs.get("lhs_batching_dimensions", ())),
                    tuple(attrs.get("rhs_batching_dimensions", ())),
                    tuple(attrs.get("lhs_contracting_dimensions", ())),
                    tuple(attrs.get("rhs_contracting_dimensions", ())))
            cached = _dot_setup.get(dkey)
            if cached is None:
                dd = _dot_dims(attrs, args[0].dim())
                rhs_ref = refs[2] if conv.kind == "dot" else refs[1]
                ws_bytes = _lib.lib().ds_dot_general_workspace_size(
                    refs[0], rhs_ref, ctypes.byref(dd), algorithm)
                if ws_bytes:  # 0: invalid; the call below reports why
                    if len(_dot_setup) > 1024:
                        _dot_setup.clear()
                    _dot_setup[dkey] = (dd, ws_bytes)
            else:
                dd, ws_bytes = cached
            ws = _workspace(ws_bytes, device, stream_ptr)
            wsp = ctypes.c_void_p(ws.data_ptr())
            if conv.kind == "dot":
                status = fn(refs[0], refs[1], refs[2], refs[3], ctypes.byref(dd), algorithm,
                            refs[4], refs[5], wsp, ws_bytes, stream)
            else:
                status = fn(refs[0], refs[1], ctypes.byref(dd), algorithm, refs[2], wsp,
                            ws_bytes, stream)
        _lib.check(status, target_name)
        return outs[0] if single else tuple(outs)

    return call


_SEQUENCE_KINDS = ("scan", "ragged", "ragged_contract")
_SCAN_TYPES = {"f64": _lib.DS_FUSED_F64, "f32": _lib.DS_FUSED_F32, "packed": _lib.DS_FUSED_PACKED}


class _Plan:
    """What a recurrence or grouped product of given shapes needs of each call:
    built on its first call, read-only afterwards."""
    __slots__ = ("fn", "dtypes", "present", "specs", "like", "table", "offsets", "workspace",
                 "attrs", "keep")


# (entry point, device index, rhs_contracting, algorithm, operand shapes...) -> _Plan
_plans: Dict[tuple, _Plan] = {}
_fast_fns: Dict[str, object] = {}


def _fast_fn(entry, operands, attrs, results):
    """The entry point with every descriptor passed as an address: three words
    (data, dims, rank) in one array for the whole call."""
    fn = _fast_fns.get(entry)
    if fn is None:
        fn = _lib.lib()[entry]  # a function object of its own
        fn.argtypes = ([ctypes.c_void_p] * operands + [ctypes.c_int32] * attrs +
                       [ctypes.c_void_p] * results +
                       [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p])
        fn.restype = ctypes.c_int
        _fast_fns[entry] = fn
    return fn


def _make_plan(sym, conv, args, specs, contracting, algorithm):
    plan = _Plan()
    L = _lib.lib()
    plan.dtypes = conv.args
    plan.present = tuple(t is not None for t in args)
    plan.keep, plan.table, plan.offsets = [], array.array("Q"), []
    for shape in [None if t is None else tuple(t.shape) for t in args] + [s.shape for s in specs]:
        plan.offsets.append(None if shape is None else 8 * len(plan.table))
        if shape is None:
            plan.table.extend((0, 0, 0))
            continue
        _, d = _lib.make_buffer(0, shape)
        plan.keep.append(d)  # the dims the plan's addresses point into
        plan.table.extend((0, ctypes.addressof(d), len(shape)))
    plan.specs = [(s.shape, s.dtype) for s in specs]
    # the operand that a result is made like (cheaper than from its shape)
    plan.like = [next((i for i, t in enumerate(args)
                       if t is not None and tuple(t.shape) == s.shape and t.dtype == s.dtype), None)
                 for s in specs]
    entry = sym
    plan.attrs = [contracting] if conv.kind == "ragged" else []
    if algorithm != _lib.DS_DOT_TENSOR_INT8:  # the entry points that take one
        entry = sym[:-4] + "_algorithm_f64" if sym.endswith("_f64") else sym + "_algorithm"
        plan.attrs.append(algorithm)
    plan.offsets[len(args):len(args)] = [None] * len(plan.attrs)

    def ref(t):
        b, d = _lib.make_buffer(t.data_ptr(), t.shape)
        plan.keep.append((b, d))
        return ctypes.byref(b)

    if conv.kind == "scan":
        plan.workspace = L.ds_linear_recurrence_workspace_size(
            ref(args[0]), _SCAN_TYPES[sym.rsplit("_", 1)[1]])
    elif conv.kind == "ragged":
        plan.workspace = L.ds_ragged_dot_algorithm_workspace_size(
            ref(args[0]), ref(args[-2]), contracting, algorithm)
    else:
        plan.workspace = L.ds_ragged_dot_contract_algorithm_workspace_size(
            ref(args[0]), ref(args[-2]), ref(args[-1]), algorithm)
    plan.fn = _fast_fn(entry, len(args), len(plan.attrs), len(specs))
    return plan


def _invoke_sequence(target_name, sym, conv, specs, args, attrs, device, out):
    """One call of a recurrence or grouped product on checked operands."""
    for i, t in enumerate(args):
        if t is not None and t.device != device:
            raise ValueError(f"{target_name} operand {i}: operands must be on one device")
    for i, t in enumerate(out or ()):
        if t.device != device:
            raise ValueError(f"{target_name} result {i}: results must be on the operands' device")
    contracting = int(attrs.get("rhs_contracting", 1))
    algorithm = int(attrs.get("algorithm", _lib.DS_DOT_TENSOR_INT8))
    key = _plan_key(sym, device.index, contracting, algorithm, args)
    plan = _plans.get(key)
    if plan is None or plan.specs != [(s.shape, s.dtype) for s in specs]:
        plan = _make_plan(sym, conv, args, specs, contracting, algorithm)
    outs = _run_plan(target_name, plan, args, device.index, out)
    if len(_plans) > 512:
        _plans.clear()
    _plans[key] = plan  # the call was accepted
    return outs


def _plan_key(sym, index, contracting, algorithm, args):
    return (sym, index, contracting, algorithm, *[None if t is None else t.shape for t in args])


def _run_plan(target_name, plan, args, index, out):
    if out is None:
        out = [torch.empty_like(args[i]) if i is not None else
               args[0].new_empty(shape, dtype=dtype)
               for i, (shape, dtype) in zip(plan.like, plan.specs)]
    table = plan.table[:]  # the call's own: (data, dims, rank) of each buffer
    at = 0
    for t in args:
        if t is not None:
            table[at] = t.data_ptr()
        at += 3
    for t in out:
        table[at] = t.data_ptr()
        at += 3
    base = table.buffer_info()[0]
    words = [None if o is None else base + o for o in plan.offsets]
    if plan.attrs:
        words[len(args):len(args) + len(plan.attrs)] = plan.attrs
    stream = _lib.current_stream_ptr(index)
    ws, wsp = None, None
    if plan.workspace:
        ws = _workspace(plan.workspace, args[0].device, stream)
        wsp = ws.data_ptr()
    _lib.check(plan.fn(*words, wsp, plan.workspace, stream), target_name)
    return out


def sequence_call(target_name, args, specs, out=None, rhs_contracting=1,
                  algorithm=_lib.DS_DOT_TENSOR_INT8):
    """ffi_call of a recurrence or grouped product without the per-call set-up:
    the plan of operands of these shapes is looked up, and operands that a
    plan's first call would accept go straight to the entry point.  `specs()`
    gives the results' ShapeDtypeStructs.  Anything else takes ffi_call, which
    checks and reports."""
    first = args[0]
    if isinstance(first, torch.Tensor) and first.is_cuda:
        index = first.get_device()
        try:
            plan = _plans.get(_plan_key(_registry[target_name], index, rhs_contracting, algorithm,
                                        args))
        except (AttributeError, TypeError):
            plan = None
        if plan is not None and out is None and torch.cuda.current_device() == index:
            for t, dt, present in zip(args, plan.dtypes, plan.present):
                if present and (t.dtype is not dt or t.get_device() != index or
                                not t.is_contiguous()):
                    break
            else:
                outs = _run_plan(target_name, plan, args, index, None)
                return outs[0] if len(outs) == 1 else tuple(outs)
    results = specs()
    attrs = {k: v for k, v in (("rhs_contracting", rhs_contracting), ("algorithm", algorithm))
             if k in CONVENTIONS[_registry[target_name]].attrs}
    return ffi_call(target_name, results if len(results) > 1 else results[0])(*args, out=out,
                                                                              **attrs)


def _dot_dims(attrs, lhs_rank) -> _lib.DsDotDims:
    lb = tuple(attrs.get("lhs_batching_dimensions", ()))
    rb = tuple(attrs.get("rhs_batching_dimensions", ()))
    lc = tuple(attrs.get("lhs_contracting_dimensions", (lhs_rank - 1,)))
    rc = tuple(attrs.get("rhs_contracting_dimensions", (len(rb),)))
    return _lib.make_dot_dims(lhs_contracting=lc, rhs_contracting=rc, lhs_batch=lb,
                              rhs_batch=rb)
