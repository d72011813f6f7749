"""Tensor-level wrappers over the HIP C ABI (HIP device tensors only; fp32, and 16-bit types where a wrapper says so;
forward only, except for the *_train functions and what they call).

Each wrapper validates shapes the way the reference does (TORCH_CHECK -> RuntimeError,
Converse2D/torch_converse2d/converse2d.cpp:167-172), makes inputs contiguous like the reference op
(:174-177), allocates outputs and workspace through torch's caching allocator and enqueues the
kernels on torch's current stream.  No CPU fallback exists here: a missing library raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
import operator
import os
import threading
from array import array
from typing import NamedTuple

import torch
from torch.multiprocessing.reductions import StorageWeakRef
from torch.overrides import _get_current_function_mode_stack
from torch.utils._device import DeviceContext

from . import _lib, composite

# The op is callable from any host thread (the reference guards its OTF cache with a mutex,
# converse2d.cpp:56,70,90): the workspace map, the plan memo and the table cache each take a lock
# around their dict updates.  Table builds run outside the locks, launches that use a stream's scratch under
# that scratch's own lock.
_ws_cache: dict = {}
_ws_lock = threading.Lock()


def _stream(dev):
    """The current stream's handle.  (torch.cuda.current_stream builds a Stream object around it: 2 us, as much
    host time as a kernel launch.)"""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _need_hip(*ts):
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("conversenet_amd HIP path needs tensors on a HIP device")
        if t.dtype != torch.float32:
            raise RuntimeError("conversenet_amd HIP path computes in float32")


class _Scratch:
    """A uint8 buffer that grows; `lock` is held while a call that uses it enqueues its kernels."""

    __slots__ = ("dev", "lock", "buf")

    def __init__(self, dev):
        self.dev, self.lock, self.buf = dev, threading.Lock(), None

    def ptr(self, nbytes):
        if nbytes == 0:
            return None
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.empty(nbytes, dtype=torch.uint8, device=self.dev)
        return self.buf.data_ptr()


def _scratch(dev, stream):
    """The scratch of the calls on a device's stream (its handle; the current one).  Its lock keeps the kernels of
    two threads' calls on one stream from alternating: one call's would overwrite what the other's still read.  A
    recorded graph gets a buffer of its own, in the graph's memory: it runs at any time, on any stream, and a kept
    buffer may be replaced by a larger one."""
    if _capturing(stream):
        return _Scratch(dev)
    key = (dev.index, stream)
    s = _ws_cache.get(key)
    if s is None:
        with _ws_lock:
            s = _ws_cache.setdefault(key, _Scratch(dev))
    return s


def release_workspace():
    with _ws_lock:
        _ws_cache.clear()


def _capturing(stream) -> bool:
    """Whether the current stream (its handle) records a graph; the null stream cannot."""
    return stream != 0 and torch._C._cuda_isCurrentStreamCapturing()


_marks: dict = {}  # (device, stream) -> event behind the latest table made there


class _Made:
    """Where the kernels that made a table were enqueued, and what other streams need before they read it."""

    __slots__ = ("dev", "stream", "event", "streams")

    def __init__(self, dev, stream):
        self.dev, self.stream = dev, stream
        self.streams = {stream}  # streams that may use the table and its memory in their own order
        # one event per stream, recorded again by each table (waiting for a later table too is no harm), without a
        # system-wide fence: writing the caches back would cost the first call on new weights 30 us
        lib = _lib.load()
        self.event = _marks.get((dev.index, stream))  # None once it is known to have passed
        if self.event is None:
            e = ctypes.c_void_p()
            with torch.cuda.device(dev):
                _lib.check(lib.cvn_event_create(ctypes.byref(e)), "transfer table")
            self.event = _marks.setdefault((dev.index, stream), e)
        _lib.check(lib.cvn_event_record(self.event, stream), "transfer table")

    def join(self, table, stream):
        """Orders the current stream (its handle) after the making of the table, and the release of the table's
        memory after what that stream has enqueued by then.  False while the making stream records a graph."""
        if self.event is not None:
            rc = _lib.load().cvn_event_join(self.event, self.stream, stream)
            if rc == _lib.CVN_ERR_UNSUPPORTED:
                return False
            _lib.check(rc, "transfer table")
        table.record_stream(torch.cuda.current_stream(self.dev))
        self.streams.add(stream)
        return True

    def finish(self):
        """Waits on the host: a stream that records a graph cannot wait for an event from outside it."""
        if self.event is not None:
            _lib.check(_lib.load().cvn_event_wait(self.event, self.stream), "transfer table")
            self.event = None


class _Entry(tuple):
    """(table, memory of psf and bias), with `made` (None without a stream)."""


class TableCache:
    """LRU cache of transfer tables, the counterpart of the reference's OTF cache (converse2d.cpp:52-102).

    Key: the psf and bias tensors (data pointer, strides and version counter), eps, the geometry, the route
    (which fixes the table's layout) and the device.  Entries hold the memory of psf and bias (detached
    views: a parameter itself drops its memory when `.data` is assigned, as Module.to does, and keeps its
    version), so a cached address cannot be reused by another tensor while the entry lives.  An in-place update
    (optimizer step, load_state_dict) bumps the version and misses; the entry of the older version is
    dropped then, so updates leave no dead tables behind.  Writes through `.data` (p.data.copy_(...),
    p.data.mul_(...)) do not bump the version counter: call torch.ops.converse2d.clear_cache() after such
    a write, as with the reference's cache, which keys on the data pointer alone.

    Callers cache only tables that can be hit again (see `cacheable`).  Bounded by the reference's
    64 entries and by bytes.

    Tables are read on any stream: a hit on another stream than the one that made the table waits for it there.
    A table made while its stream records a graph exists once the graph has run, so it is not kept; one from
    before that the graph reads stays until the psf's memory is released (the graph goes on reading it after an
    update of the parameters and clear_cache: record it again then).  At most max_entries tables stay that way;
    past that, a graph makes its own."""

    def __init__(self, max_entries=64, max_bytes=4 << 30):
        from collections import OrderedDict

        self.entries = OrderedDict()
        self._lock = threading.RLock()
        self.latest = {}  # key without version counters -> full key
        self.max_entries = max_entries
        self.max_bytes = max_bytes
        self.bytes = 0
        self.hits = 0
        self.misses = 0
        self.recorded = []  # (psf storage, table) read by recorded graphs

    @staticmethod
    def _stem(key):
        return key[:2] + key[3:4] + key[5:]

    def _keep_recorded(self, e):  # caller holds self._lock
        self.recorded = [r for r in self.recorded if not r[0].expired()]
        if any(t is e[0] for _, t in self.recorded):
            return True
        if len(self.recorded) >= self.max_entries or sum(t.numel() for _, t in self.recorded) > self.max_bytes:
            return False
        self.recorded.append((StorageWeakRef(e[1][0].untyped_storage()), e[0]))
        return True

    def _usable(self, e, stream):  # caller holds self._lock
        if _capturing(stream):
            e.made.finish()
            return self._keep_recorded(e)
        return stream in e.made.streams or e.made.join(e[0], stream)

    def get(self, key, stream=None):
        """The table of `key` or None.  stream: the current stream's handle, where the table is to be read."""
        with self._lock:
            e = self.entries.get(key)
            if e is None or not (e.made is None or stream is None or self._usable(e, stream)):
                self.misses += 1
                return None
            self.entries.move_to_end(key)
            self.hits += 1
            return e[0]

    def _drop(self, key):  # caller holds self._lock
        t, _ = self.entries.pop(key)
        self.bytes -= t.numel()
        stem = self._stem(key)
        if self.latest.get(stem) == key:
            del self.latest[stem]

    def put(self, key, table, refs, stream=None):
        """Keeps `table`.  stream: the current stream's handle, where its kernels have been enqueued."""
        if stream is not None and _capturing(stream):
            return
        e = _Entry((table, tuple(t.detach() for t in refs)))
        e.made = None if stream is None else _Made(table.device, stream)
        with self._lock:
            old = self.latest.get(self._stem(key))
            if old is not None and old in self.entries:
                self._drop(old)  # the same tensors at an older version: never hit again
            prev = self.entries.pop(key, None)
            if prev is not None:  # another thread built the same table meanwhile: keep one copy
                self.bytes -= prev[0].numel()
            self.entries[key] = e
            self.latest[self._stem(key)] = key
            self.bytes += table.numel()
            while self.entries and (len(self.entries) > self.max_entries or self.bytes > self.max_bytes):
                self._drop(next(iter(self.entries)))

    def clear(self):
        with self._lock:
            self.entries.clear()
            self.latest.clear()
            self.bytes = 0


table_cache = TableCache()


def cacheable(weight, bias) -> bool:
    """Whether a table for (weight, bias) can be hit by a later call: not for inference tensors (no
    version counter; in inference mode they are fresh activations), and not while autograd tracks the
    parameters (an optimizer step changes them before the next call; the reference bypasses its cache
    then, converse2d.cpp:60,68,88)."""
    for t in (weight, bias):
        if t.is_inference() or (torch.is_grad_enabled() and t.requires_grad):
            return False
    return True


def _cache_key(kind, weight, bias, eps, geo, route, dev):
    # with the strides of a view: a transposed or expanded one starts at its base's address and shares its version
    return (kind, weight.data_ptr(), weight._version, bias.data_ptr(), bias._version, float(eps), geo, route,
            dev.index, None if weight.is_contiguous() else weight.stride(),
            None if bias.is_contiguous() else bias.stride())


# os.environ's own mapping: a name that is not set costs 0.6 us through os.environ, which raises for it twice
_ENV = os.environ._data
_plan_memo: dict = {}
_supported_memo: dict = {}  # the library's answers by geometry, as in _plan_memo
_plan_lock = threading.Lock()


def _module_plan(lib, B, C, H, W, pb, kh, kw, s, p):
    """(route, table bytes, scratch bytes) of a module-level call: the library's answers depend only on
    the geometry and CVN_DISABLE_FUSED, so they are asked once per geometry (three queries cost about as
    much host time as a small layer's kernels)."""
    key = (B, C, H, W, pb, kh, kw, s, p, _ENV.get(b"CVN_DISABLE_FUSED"))
    plan = _plan_memo.get(key)
    if plan is None:
        route = lib.cvn_converse2d_route(B, C, H, W, pb, kh, kw, s, p)
        if route < 0:
            _lib.check(route, "converse2d_fused")
        plan = (route, lib.cvn_converse2d_table_bytes(B, C, H, W, pb, kh, kw, s, p, route),
                lib.cvn_converse2d_scratch_bytes(B, C, H, W, pb, kh, kw, s, p, route))
        with _plan_lock:
            if len(_plan_memo) >= 1024:
                _plan_memo.clear()
            _plan_memo[key] = plan
    return plan


def module_route(shape, weight, scale, padding):
    """The library's route (_lib.ROUTE_*) for a module-level call on an input of `shape` (B, C, H, W)."""
    B, C, H, W = (int(v) for v in shape)
    return _module_plan(_lib.load(), B, C, H, W, int(weight.shape[0]), int(weight.shape[2]), int(weight.shape[3]),
                        int(scale), int(padding))[0]


def converse2d_fused(x, weight, bias, scale=1, padding=2, padding_mode="circular", eps=1e-5, act=None,
                     cache=True):
    """Converse2D.forward (util_converse.py:142-192) in one library call: pad, solve, crop.

    x (B,C,H,W); weight (1,C,kh,kw) or (B,C,kh,kw) (per-sample psf, as ConvReverseDataNet);
    bias (1,C,1,1) or (C,).  act='gelu' applies exact GELU to the output on store.  cache=True keeps
    the transfer table of a shared psf (psf batch 1) for reuse while weight and bias are unchanged
    (version-checked); per-sample psfs are activations that change every call and are not cached."""
    lib = _lib.load()
    _need_hip(x, weight, bias)
    if x.dim() != 4:
        raise RuntimeError("x must be (B,C,H,W)")
    B, C, H, W = x.shape
    if weight.dim() != 4 or weight.shape[1] != C or weight.shape[0] not in (1, B):
        raise RuntimeError("weight must be (1,C,kh,kw) or (B,C,kh,kw)")
    if bias.numel() != C:
        raise RuntimeError("bias must hold C values")
    if padding_mode not in _lib.PAD_MODES:
        raise ValueError(f"unknown padding_mode {padding_mode!r}")
    s = int(scale)
    if s < 1:
        raise RuntimeError("scale must be >= 1")
    kh, kw = int(weight.shape[2]), int(weight.shape[3])
    pb = int(weight.shape[0])
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    dev = x.device
    out = torch.empty((B, C, H * s, W * s), dtype=torch.float32, device=dev)
    if B == 0:
        return out
    p = int(padding)
    route, tb, sb = _module_plan(lib, B, C, H, W, pb, kh, kw, s, p)
    st = _stream(dev)
    key = None
    table = None
    if cache and pb == 1 and cacheable(weight, bias):
        key = _cache_key("module", weight, bias, eps, (C, H, W, kh, kw, s, p), route, dev)
        table = table_cache.get(key, st)
    if table is None:
        wc = weight.contiguous()
        bc = bias.contiguous()
        table = torch.empty(tb, dtype=torch.uint8, device=dev)
        _lib.check(lib.cvn_converse2d_table_f32(wc.data_ptr(), pb, kh, kw, bc.data_ptr(), float(eps), B, C, H, W,
                                                s, p, route, table.data_ptr(), tb, st), "converse2d transfer table")
        if key is not None:
            table_cache.put(key, table, (weight, bias), st)
    ws = _scratch(dev, st)
    with ws.lock:
        rc = lib.cvn_converse2d_apply_f32(
            x.data_ptr(), B, C, H, W, pb, kh, kw, s, p, _lib.PAD_MODES[padding_mode],
            _lib.ACT_GELU if act == "gelu" else _lib.ACT_NONE, route, table.data_ptr(), tb, ws.ptr(sb), sb,
            out.data_ptr(), st)
    _lib.check(rc, "converse2d_fused")
    return out


def supported(x, weight, scale, padding, grad_x=False, grad_weight=False, shape=None) -> bool:
    """Whether the library's forward (and the requested backward) serves this geometry
    (cvn_converse2d_supported); shapes it does not serve go to the PyTorch composition.  shape
    (B, C, H, W) stands in for x's shape when given."""
    lib = _lib.load()
    if weight.dim() != 4 or (shape is None and x.dim() != 4):
        return False
    B, C, H, W = shape if shape is not None else x.shape
    pb, _, kh, kw = weight.shape
    key = (B, C, H, W, pb, kh, kw, int(scale), int(padding), bool(grad_x), bool(grad_weight),
           _ENV.get(b"CVN_DISABLE_FUSED"))
    ok = _supported_memo.get(key)
    if ok is None:
        ok = lib.cvn_converse2d_supported(*key[:9], int(key[9]), int(key[10])) == _lib.CVN_OK
        with _plan_lock:
            if len(_supported_memo) >= 1024:
                _supported_memo.clear()
            _supported_memo[key] = ok
    return ok


def op_supported(x, x0, weight, scale) -> bool:
    """Whether the library's operator path serves this call (its table and scratch queries are
    non-zero for the geometry); shapes it does not serve go to the PyTorch composition.  Malformed
    arguments also answer False here and are then rejected by the composition's checks."""
    if x.dim() != 4 or x0.dim() != 4 or weight.dim() != 4:
        return False
    s = int(scale)
    B, C, h, w = (int(v) for v in x.shape)
    if s < 1 or tuple(x0.shape) != (B, C, h * s, w * s) or weight.shape[0] != 1 or weight.shape[1] != C:
        return False
    if B == 0:
        return True  # an empty batch returns its empty output without a launch (converse2d_op)
    if (s == 1 and x0.data_ptr() == x.data_ptr() and x0.stride() == x.stride() and B > 0
            and supported(x, weight, 1, 0)):
        return True  # served by the module route on the padded plane (converse2d_op)
    lib = _lib.load()
    kh, kw = int(weight.shape[2]), int(weight.shape[3])
    return (lib.cvn_converse2d_op_table_bytes(C, h, w, kh, kw, s) > 0
            and lib.cvn_converse2d_op_scratch_bytes(B, C, h, w, s) > 0)


def converse2d_backward(grad_out, x, weight, bias, scale=1, padding=2, padding_mode="circular", eps=1e-5,
                        need_x=True, need_weight=True, need_bias=True):
    """Gradients of Converse2D.forward (util_converse.py:142-192) in one library call: returns
    (grad_x, grad_weight, grad_bias), None where not requested.  grad_out (B,C,H*s,W*s); weight
    (1 or B, C, kh, kw); bias (1,C,1,1) or (C,)."""
    lib = _lib.load()
    _need_hip(grad_out, x, weight, bias)
    B, C, H, W = x.shape
    s, p = int(scale), int(padding)
    if tuple(grad_out.shape) != (B, C, H * s, W * s):
        raise RuntimeError("grad_out must be (B,C,H*scale,W*scale)")
    if weight.dim() != 4 or weight.shape[1] != C or weight.shape[0] not in (1, B):
        raise RuntimeError("weight must be (1,C,kh,kw) or (B,C,kh,kw)")
    if padding_mode not in _lib.PAD_MODES:
        raise ValueError(f"unknown padding_mode {padding_mode!r}")
    kh, kw = int(weight.shape[2]), int(weight.shape[3])
    pb = int(weight.shape[0])
    dev = x.device
    go = grad_out.contiguous()
    xc = x.contiguous()
    wc = weight.contiguous()
    bc = bias.contiguous()
    gx = torch.empty((B, C, H, W), dtype=torch.float32, device=dev) if need_x else None
    gw = torch.empty((pb, C, kh, kw), dtype=torch.float32, device=dev) if need_weight else None
    gb = torch.empty((C,), dtype=torch.float32, device=dev) if need_bias else None
    if B == 0 or not (need_x or need_weight or need_bias):
        for t in (gw, gb):
            if t is not None:
                t.zero_()
        return gx, gw, gb.reshape(bias.shape) if gb is not None else None
    nb = lib.cvn_converse2d_bwd_workspace(B, C, H, W, pb, kh, kw, s, p)
    if nb == 0:
        _lib.check(_lib.CVN_ERR_ARG, "converse2d_backward")
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    st = _stream(dev)
    ws = _scratch(dev, st)
    with ws.lock:
        rc = lib.cvn_converse2d_bwd_f32(go.data_ptr(), xc.data_ptr(), B, C, H, W, wc.data_ptr(), pb, kh, kw,
                                        bc.data_ptr(), float(eps), s, p, _lib.PAD_MODES[padding_mode], ptr(gx),
                                        ptr(gw), ptr(gb), ws.ptr(nb), nb, st)
    _lib.check(rc, "converse2d_backward")
    return gx, gw, gb.reshape(bias.shape) if gb is not None else None


class Converse2DFunction(torch.autograd.Function):
    """Converse2D.forward with the library's forward and backward kernels (the reference gets its
    gradients from autograd through the composite op, converse2d.cpp:223-227)."""

    @staticmethod
    def forward(ctx, x, weight, bias, scale, padding, padding_mode, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.cfg = (scale, padding, padding_mode, eps)
        # the parameters change between training steps, so their tables are not cached
        return converse2d_fused(x, weight, bias.reshape(-1), scale, padding, padding_mode, eps, cache=False)

    @staticmethod
    def backward(ctx, grad_out):
        x, weight, bias = ctx.saved_tensors
        s, p, mode, eps = ctx.cfg
        nx, nw, nb = ctx.needs_input_grad[:3]
        gx, gw, gb = converse2d_backward(grad_out, x, weight, bias, s, p, mode, eps, nx, nw, nb)
        return gx, gw, gb, None, None, None, None


def converse2d_train(x, weight, bias, scale=1, padding=2, padding_mode="circular", eps=1e-5):
    """Differentiable Converse2D forward on the HIP kernels (forward and backward)."""
    return Converse2DFunction.apply(x, weight, bias, scale, padding, padding_mode, eps)


def converse2d_op(x, x0, weight, bias, scale, eps=1e-5, cache=True):
    """The reference op (converse2d.cpp:165-209): x padded (B,C,h,w), x0 (B,C,h*s,w*s) arbitrary;
    returns the uncropped (B,C,h*s,w*s) solution.  The op table (OTF and alias-class terms) is cached
    per (psf, bias, eps, geometry) like the reference's OTF (p2o_cached, converse2d.cpp:58-102)."""
    lib = _lib.load()
    composite.check_op_args(x, x0, weight, bias, scale)
    s = int(scale)
    _need_hip(x, x0, weight, bias)
    B, C, h, w = x.shape
    if tuple(x0.shape) != (B, C, h * s, w * s) or weight.shape[1] != C or bias.shape[1] != C:
        raise RuntimeError("shape mismatch between x, x0, weight and bias")
    if (s == 1 and x0.data_ptr() == x.data_ptr() and x0.stride() == x.stride() and B > 0
            and supported(x, weight, 1, 0)):
        # x0 is x, as the reference module passes it at scale 1 (util_converse.py:166): then
        # X0 = Y and the solve is the module's X = Y (conj K + lambda) / (|K|^2 + lambda) on the
        # given (already padded) plane, one forward and one inverse transform instead of two and one
        return converse2d_fused(x, weight, bias.reshape(-1), 1, 0, "constant", eps, cache=cache)
    x, x0 = x.contiguous(), x0.contiguous()
    dev = x.device
    out = torch.empty((B, C, h * s, w * s), dtype=torch.float32, device=dev)
    if B == 0:
        return out
    kh, kw = int(weight.shape[2]), int(weight.shape[3])
    tb = lib.cvn_converse2d_op_table_bytes(C, h, w, kh, kw, s)
    sb = lib.cvn_converse2d_op_scratch_bytes(B, C, h, w, s)
    if tb == 0 or sb == 0:
        _lib.check(lib.cvn_converse2d_op_f32(None, None, B, C, h, w, None, kh, kw, None, float(eps), s, None, None,
                                             0, None), "converse2d_op")
    st = _stream(dev)
    key = None
    table = None
    if cache and cacheable(weight, bias):
        key = _cache_key("op", weight, bias, eps, (C, h, w, kh, kw, s), 0, dev)
        table = table_cache.get(key, st)
    if table is None:
        wc, bc = weight.contiguous(), bias.contiguous()
        table = torch.empty(tb, dtype=torch.uint8, device=dev)
        _lib.check(lib.cvn_converse2d_op_table_f32(wc.data_ptr(), kh, kw, bc.data_ptr(), float(eps), C, h, w, s,
                                                   table.data_ptr(), tb, st), "converse2d op table")
        if key is not None:
            table_cache.put(key, table, (weight, bias), st)
    ws = _scratch(dev, st)
    with ws.lock:
        rc = lib.cvn_converse2d_op_apply_f32(x.data_ptr(), x0.data_ptr(), B, C, h, w, s, table.data_ptr(), tb,
                                             ws.ptr(sb), sb, out.data_ptr(), st)
    _lib.check(rc, "converse2d_op")
    return out


def converse2d_fwd_oneshot(x, weight, bias, scale=1, padding=2, padding_mode="circular", eps=1e-5, act=None):
    """cvn_converse2d_fwd_f32: the whole module-level forward (table and apply) in one library call, on
    the route the library picks, with one caller workspace."""
    lib = _lib.load()
    _need_hip(x, weight, bias)
    B, C, H, W = x.shape
    s, p = int(scale), int(padding)
    kh, kw, pb = int(weight.shape[2]), int(weight.shape[3]), int(weight.shape[0])
    x, wc, bc = x.contiguous(), weight.contiguous(), bias.contiguous()
    if x.data_ptr() % 16:  # the fused route reads rows as 16-byte vectors
        x = x.clone()
    out = torch.empty((B, C, H * s, W * s), dtype=torch.float32, device=x.device)
    nb = lib.cvn_converse2d_fwd_workspace(B, C, H, W, pb, kh, kw, s, p)
    st = _stream(x.device)
    ws = _scratch(x.device, st)
    with ws.lock:
        rc = lib.cvn_converse2d_fwd_f32(x.data_ptr(), B, C, H, W, wc.data_ptr(), pb, kh, kw, bc.data_ptr(), float(eps),
                                        s, p, _lib.PAD_MODES[padding_mode],
                                        _lib.ACT_GELU if act == "gelu" else _lib.ACT_NONE, out.data_ptr(),
                                        ws.ptr(max(nb, 1)), nb, st)
    _lib.check(rc, "converse2d_fwd")
    return out


def layernorm_cf(x, weight, bias, eps):
    """LayerNorm(data_format='channels_first') (util_converse.py:63-68)."""
    lib = _lib.load()
    _need_hip(x, weight, bias)
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    B, C = x.shape[:2]
    HW = x[0, 0].numel() if B > 0 else 0
    y = torch.empty_like(x)
    _lib.check(lib.cvn_layernorm_cf_f32(x.data_ptr(), B, C, HW, weight.data_ptr(), bias.data_ptr(), float(eps),
                                        y.data_ptr(), _stream(x.device)), "layernorm_cf")
    return y


def _ptrs(keep, *ts):
    """Addresses of contiguous tensors (None for None).  Copies of others go to `keep`, which the caller holds until
    the call has enqueued its kernels: a copy that is dropped before then gives its memory to the next copy or
    output."""
    out = []
    for t in ts:
        if t is not None and not t.is_contiguous():
            t = t.contiguous()
            keep.append(t)
        out.append(None if t is None else t.data_ptr())
    return out


def conv1x1(x, weight, bias=None, act=None, residual=None, res_scale=None, ln=None, out=None):
    """act(W x + b) [then res_scale * . + residual]; nn.Conv2d(cin, cout, 1) semantics.
    ln=(ln_weight, ln_bias, eps) applies channels-first LayerNorm to x first (fused prologue)."""
    lib = _lib.load()
    _need_hip(x, weight, bias, residual, res_scale)
    x = x.contiguous()
    B, Cin, H, W = x.shape
    Cout = weight.shape[0]
    if weight.numel() != Cout * Cin:
        raise RuntimeError("weight does not match input channels")
    y = out if out is not None else torch.empty((B, Cout, H, W), dtype=torch.float32, device=x.device)
    keep = []
    wptr, bptr, rptr, sptr = _ptrs(keep, weight, bias, residual, res_scale)
    a = _lib.ACT_GELU if act == "gelu" else _lib.ACT_NONE
    st = _stream(x.device)
    if ln is None:
        rc = lib.cvn_conv1x1_f32(x.data_ptr(), B, Cin, H * W, wptr, bptr, Cout, a, rptr, sptr, y.data_ptr(), st)
    else:
        rc = lib.cvn_ln_conv1x1_f32(x.data_ptr(), B, Cin, H * W, *_ptrs(keep, *ln[:2]), float(ln[2]), wptr, bptr, Cout,
                                    a, rptr, sptr, y.data_ptr(), st)
    _lib.check(rc, "conv1x1")
    return y


def ln_mlp_residual(x, ln_w, ln_b, ln_eps, w1, b1, w2, b2, res_scale=None, out=None):
    """x + res_scale * (W2 GELU(W1 LN(x) + b1) + b2): ConverseBlock.conv2 plus its residual."""
    lib = _lib.load()
    _need_hip(x, w1, b1, w2, b2, res_scale)
    x = x.contiguous()
    B, C, H, W = x.shape
    keep = []
    y = out if out is not None else torch.empty_like(x)
    lw, lb, w1_, b1_, w2_, b2_, sp = _ptrs(keep, ln_w, ln_b, w1, b1, w2, b2, res_scale)
    rc = lib.cvn_ln_mlp_residual_f32(x.data_ptr(), B, C, H * W, lw, lb, float(ln_eps), w1_, b1_, w1.shape[0], w2_, b2_,
                                     sp, y.data_ptr(), _stream(x.device))
    _lib.check(rc, "ln_mlp_residual")
    return y


TAIL_SHAPES = {(128, 64, 128)}  # (Ct, C, Cmid) of cvn_conv_ln_mlp_residual_f32


def conv_ln_mlp_residual(t, x, w0, b0, ln_w, ln_b, ln_eps, w1, b1, w2, b2, res_scale1=None, res_scale2=None,
                         out=None, head=None, t_act=None):
    """ConverseBlock tail: y' = x + res_scale1 (W0 a(t) + b0); y = y' + res_scale2 (W2 GELU(W1 LN(y') + b1) + b2),
    a(t) = GELU(t) for t_act='gelu' (t the Converse2D output before the block's GELU), else t.
    With head = (ln_w, ln_b, ln_eps, w, b) of the next block, also returns its Converse2D input
    GELU(w LN(y) + b): (y, t_next); otherwise y."""
    lib = _lib.load()
    _need_hip(t, x, w0, b0, w1, b1, w2, b2, res_scale1, res_scale2)
    t = t.contiguous()
    x = x.contiguous()
    B, Ct, H, W = t.shape
    C = x.shape[1]
    y = out if out is not None else torch.empty_like(x)
    act = _lib.ACT_GELU if t_act == "gelu" else _lib.ACT_NONE
    keep = []
    w0_, b0_, s1, lw, lb, w1_, b1_, w2_, b2_, s2 = _ptrs(keep, w0, b0, res_scale1, ln_w, ln_b, w1, b1, w2, b2, res_scale2)
    common = (t.data_ptr(), act, B, Ct, H * W, w0_, b0_, s1, x.data_ptr(), C, lw, lb, float(ln_eps), w1_, b1_,
              w1.shape[0], w2_, b2_, s2, y.data_ptr())
    if head is None:
        _lib.check(lib.cvn_conv_ln_mlp_residual_f32(*common, _stream(x.device)), "conv_ln_mlp_residual")
        return y
    hw, hb, heps, wh, bh = head
    _need_hip(wh, bh)
    hw_, hb_, wh_, bh_ = _ptrs(keep, hw, hb, wh, bh)
    tn = torch.empty((B, wh.shape[0], H, W), device=x.device, dtype=x.dtype)
    _lib.check(lib.cvn_conv_ln_mlp_head_f32(*common, hw_, hb_, float(heps), wh_, bh_, tn.data_ptr(), _stream(x.device)),
               "conv_ln_mlp_head")
    return y, tn


def _on(dev):
    """Makes a tensor's device current for the launches on its stream."""
    return _NO_SWITCH if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


_NO_SWITCH = contextlib.nullcontext()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _param32(keep, t, C, index, what):
    """Address of a parameter's C values in float32 (None for None); copies go to `keep`, as in _ptrs."""
    if t is None:
        return None
    if t.get_device() != index or t.numel() != C or t.dtype not in _lib.TYPES:
        raise RuntimeError(f"{what} must hold {C} values on the device of x")
    if t.dtype is not torch.float32 or not t.is_contiguous():
        t = t.to(torch.float32).contiguous()
        keep.append(t)
    at = t.data_ptr()
    if not at and C:  # (the library would take it for none)
        raise RuntimeError(f"{what} stands for other tensors: it has no memory to compute on")
    return at


def _gate_kind(h, gate):
    if gate is None:
        return _lib.GATE_NONE
    if gate.shape == h.shape:
        return _lib.GATE_FULL
    if tuple(gate.shape) in (tuple(h.shape[:2]), tuple(h.shape[:2]) + (1,) * (h.dim() - 2)):
        return _lib.GATE_SAMPLE
    raise RuntimeError("gate must have the branch's shape, or (B,C) or (B,C,1,..) for a factor per sample and channel")


_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack
_tracing_state = torch._C._get_tracing_state


def _pre_dispatch() -> int:
    return torch._ops._len_torch_dispatch_stack_pre_dispatch() if _function_modes() else 0


def observed() -> bool:
    """Whether a mode of the caller's sees torch's operations: it would miss those that the library stands for.  (A
    default device is such a mode, and changes nothing here.)"""
    if _dispatch_modes():
        return True
    return _function_modes() > 0 and any(type(m) is not DeviceContext for m in _get_current_function_mode_stack())


def _untraced(what):
    """Refuses a call that is being recorded as torch operations: the library's kernels are none, and the recorded graph
    would return its outputs as they were allocated."""
    if _tracing_state() is not None or _pre_dispatch() or (
            _dispatch_modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        raise RuntimeError(f"{what} cannot be traced as torch operations")


def _norm_args(x, h, gate):
    """Checks the large arguments of a residual_norm call: ((B, C, HW, kind of gate), device index)."""
    if _dispatch_modes() or _function_modes() or _tracing_state() is not None:
        _untraced("residual_norm")
    index = x.get_device()
    for t in (x, h, gate):
        if t is not None and (t.get_device() != index or index < 0 or t.dtype not in _lib.TYPES):
            raise RuntimeError("residual_norm needs float32, bfloat16 or float16 tensors on one HIP device")
    shape = x.shape
    if len(shape) < 2 or shape[1] < 1:
        raise RuntimeError("x must be (B,C,*) with channels")
    if h is not None:
        if h.shape != shape:
            raise RuntimeError("x and the branch must have one shape")
        if h.dtype is not x.dtype and x.dtype is not torch.float32:
            raise RuntimeError("x and the branch must have one type, or x float32 and the branch a 16-bit type")
        if gate is not None and gate.dtype is not h.dtype:
            raise RuntimeError("gate must have the branch's type")
    return (shape[0], shape[1], math.prod(shape[2:]), _gate_kind(h, gate)), index


def _residual_norm(x, h, norm, res_scale, gate, post, need_stats, copy=False):
    """The launch behind residual_norm, on contiguous x, h and gate: (r, y, stats, what _norm_args gave, whether the
    parameters were read where they are), None for what there is not.  copy: r is a copy of x where there is no h."""
    lib = _lib.load()
    geo, index = _norm_args(x, h, gate)
    B, C, HW, kind = geo
    keep = []
    s = _param32(keep, res_scale, C, index, "res_scale")
    nw = nb = pw = pb = r = y = stats = None
    neps = peps = 0.0
    if norm is not None:
        nw, nb = _param32(keep, norm[0], C, index, "norm weight"), _param32(keep, norm[1], C, index, "norm bias")
        neps = float(norm[2])
        y = torch.empty_like(x)
    if post is not None:
        pw, pb = _param32(keep, post[0], C, index, "branch norm"), _param32(keep, post[1], C, index, "branch norm")
        peps = float(post[2])
    if h is not None or copy:
        r = torch.empty_like(x)
    dev = x.device
    if need_stats and (norm is not None or post is not None):
        stats = torch.empty((2 if post is None else 4, B * HW), dtype=torch.float32, device=dev)
    with _on(dev):
        rc = lib.cvn_residual_norm_fwd(x.data_ptr(), _lib.TYPES[x.dtype], _ptr(h), _lib.TYPES[(x if h is None else h).dtype],
                                       B, C, HW, s, _ptr(gate), kind, pw, pb, peps, nw, nb, neps, _ptr(r), _ptr(y),
                                       _ptr(stats), _stream(dev))
    _lib.check(rc, "residual_norm")
    return r, y, stats, geo, not keep


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def residual_norm(x, h, norm=None, res_scale=None, gate=None, post=None):
    """A block's scaled residual and the norms before and after its branch, in one pass:
    r = x + res_scale * gate * P(h), y = N(r); returns (r, y), y None without norm.

    x, h (B,C,*), channels first, of one type, or a 16-bit branch h on a float32 x; r and y have x's type.
    norm, post: (weight, bias, eps) of channels-first LayerNorms of r and of the branch (P(h) = h without post);
    res_scale: C values (ConverseBlockAlphaVariant's alphas, util_converse.py:321-322); gate: a factor per element
    (h's shape) or per sample and channel ((B,C) or (B,C,1,1)), of h's type.  Computed in float32, each output
    rounded once: y is the norm of r before its rounding.  For gradients see residual_norm_train."""
    if h is None:
        raise RuntimeError("residual_norm needs a branch")
    return _residual_norm(_contiguous(x), _contiguous(h), norm, res_scale, _contiguous(gate), post, False)[:2]


@functools.lru_cache(maxsize=1024)
def _norm_workspace(geo):
    """Bytes of scratch of a backward of this geometry (the library's answer depends on nothing else)."""
    return _lib.load().cvn_residual_norm_bwd_workspace(*geo)


def _residual_norm_backward(gr, gy, base, h, stats, norm_w, nb_shape, res_scale, gate, post_w, post_b, geo, shape, x_dtype,
                            h_dtype, need, direct=False):
    """The launches behind residual_norm_backward, on arguments that a forward has checked; direct: it read the
    parameters where they are."""
    lib = _lib.load()
    B, C, HW, kind = geo
    nx, nh, ns, ng, npw, npb, nnw, nnb = need
    gr, gy = _contiguous(gr), _contiguous(gy) if norm_w is not None else None
    some = gr if gr is not None else gy
    dev = some.device
    keep = []
    f32 = torch.float32

    def like(t, wanted):  # (empty_like takes half the time of empty)
        if not wanted or t is None:
            return None
        return torch.empty_like(t) if direct else torch.empty(t.shape, dtype=f32, device=dev)

    plain = res_scale is None and gate is None and post_w is None  # then the branch's gradient is x's
    gx = gh = gnw = gnb = out_x = out_h = None
    nh = nh and h_dtype is not None
    same = nh and plain and h_dtype is x_dtype
    if gy is not None:
        if nx or same:
            gx = out_x = torch.empty_like(some)
        gnw = like(norm_w, nnw)
        if nnb:  # (empty_like where it can be)
            gnb = like(norm_w, True) if norm_w.shape == nb_shape else torch.empty(nb_shape, dtype=f32, device=dev)
    else:  # x's gradient is r's
        gx = gr
        if norm_w is not None:  # y was not used
            gnw, gnb = (torch.zeros(t, dtype=f32, device=dev) if w else None
                        for t, w in ((norm_w.shape, nnw), (nb_shape, nnb)))
    if same:
        gh = gx
    elif nh and plain and gy is None:
        gh = gr.to(h_dtype)
    elif nh:
        gh = out_h = torch.empty_like(h) if h is not None else torch.empty(shape, dtype=h_dtype, device=dev)
    gs, gpw, gpb = like(res_scale, ns), like(post_w, npw), like(post_b, npb)
    gg = torch.empty_like(gate) if ng and gate is not None else None
    if gy is not None or out_h is not None or gs is not None or gg is not None or gpw is not None or gpb is not None:
        params = (res_scale, post_w, post_b, None if gy is None else norm_w)
        if direct:
            s, pw, pb, nw = map(_ptr, params)
        else:
            s, pw, pb, nw = (_param32(keep, t, C, dev.index, "a parameter") for t in params)
        nbytes = _norm_workspace(geo)
        st = _stream(dev)
        ws = _scratch(dev, st)
        with _on(dev), ws.lock:
            rc = lib.cvn_residual_norm_bwd(
                _ptr(gr), _ptr(gy), None if gy is None else base.data_ptr(), _lib.TYPES[x_dtype], _ptr(h),
                _lib.TYPES[h_dtype or x_dtype], B, C, HW, s, _ptr(gate), kind, pw, pb, nw, _ptr(stats), _ptr(out_x),
                _ptr(out_h), _ptr(gg), _ptr(gs), *((None, None) if gy is None else (_ptr(gnw), _ptr(gnb))), _ptr(gpw),
                _ptr(gpb), ws.ptr(nbytes), nbytes, st)
        _lib.check(rc, "residual_norm_backward")
    return (gx if nx else None), gh, gs, gg, gpw, gpb, gnw, gnb


def residual_norm_backward(grad_r, grad_y, base, h, stats, norm_weight=None, res_scale=None, gate=None, post=None,
                           h_dtype=None, need=(True,) * 8):
    """Gradients of residual_norm in one call: (x, h, res_scale, gate, post weight, post bias, norm weight, norm bias),
    None where not asked for by `need` or not given; those of parameters in float32.

    grad_r, grad_y: gradients of r and y (None: zero).  base: the forward's r where x is float32, x itself where it
    is a 16-bit type (there the norm is that of r before its rounding), or None without norm_weight.  h may be None
    where x is float32 and there is no scale, gate and post: its gradient is x's, of type h_dtype.  stats: mean and
    1 / deviation of r, and with post of h, float32 (2 or 4, B HW), as residual_norm_stats gives them."""
    ref = next((t for t in (base, grad_r, grad_y) if t is not None), None)
    if ref is None or (norm_weight is None and grad_r is None) or (norm_weight is not None and base is None):
        raise RuntimeError("residual_norm_backward needs a gradient, and what its norm was of")
    if h is not None:
        h_dtype = h.dtype
    elif res_scale is not None or gate is not None or post is not None or (ref.dtype != torch.float32 and (
            h_dtype or (grad_r is not None and grad_y is not None))):
        raise RuntimeError("residual_norm_backward needs the branch")
    h, gate = _contiguous(h), _contiguous(gate)
    geo, index = _norm_args(ref, h, gate)
    for t in (grad_r, grad_y):
        if t is not None and (t.shape != ref.shape or t.dtype != ref.dtype or t.get_device() != index):
            raise RuntimeError("gradients must match r and y")
    if (norm_weight is not None or post is not None) and (
            stats is None or tuple(stats.shape) != (2 if post is None else 4, geo[0] * geo[2])
            or not stats.is_contiguous() or stats.dtype != torch.float32 or stats.get_device() != index):
        raise RuntimeError("stats must be the forward's")
    if grad_r is None and grad_y is None:
        raise RuntimeError("residual_norm_backward needs a gradient")
    pw, pb = (None, None) if post is None else post[:2]
    return _residual_norm_backward(grad_r, grad_y, _contiguous(base), h, stats, norm_weight,
                                   None if norm_weight is None else norm_weight.shape, res_scale, gate, pw, pb, geo, ref.shape,
                                   ref.dtype, h_dtype, need)


def residual_norm_stats(x, h, norm=None, res_scale=None, gate=None, post=None):
    """residual_norm with what residual_norm_backward needs of it: (r, y, stats).  h may be None: y = N(x), r None."""
    if h is None and (res_scale is not None or gate is not None or post is not None or norm is None):
        raise RuntimeError("without a branch there is only the norm of x")
    return _residual_norm(_contiguous(x), _contiguous(h), norm, res_scale, _contiguous(gate), post, True)[:3]


def _in_memory(t):
    """Whether a gradient (None: true) is a plain tensor: one that stands for many, or for none yet, has no address."""
    try:
        return t is None or type(t) in (torch.Tensor, torch.nn.Parameter) and t.data_ptr() is not None
    except RuntimeError:
        return False


class ResidualNormFunction(torch.autograd.Function):
    """residual_norm (h None: LayerNorm alone) with the library's forward and backward kernels.  A backward that is
    itself to be differentiated, mapped over many gradients at once or seen by a dispatch mode (a tracer among them) runs as a
    composition of torch operations."""

    @staticmethod
    def forward(ctx, x, h, res_scale, gate, post_w, post_b, norm_w, norm_b, post_eps, norm_eps, copy=False):
        # x, h and gate are contiguous: a copy made here would not be the caller's in a differentiated backward
        ctx.set_materialize_grads(False)
        post = None if post_w is None else (post_w, post_b, post_eps)
        norm = None if norm_w is None else (norm_w, norm_b, norm_eps)
        r, y, stats, geo, direct = _residual_norm(x, h, norm, res_scale, gate, post, True, copy)
        f32 = x.dtype is torch.float32
        keep_h = h is not None and not (f32 and res_scale is None and gate is None and post is None)
        base = None if norm is None else (r if copy or (h is not None and f32) else x)
        # (of the norm's bias no value is needed: it may change before the backward)
        ctx.save_for_backward(base, h if keep_h else None, res_scale, gate, post_w, post_b, norm_w, stats)
        ctx.cfg = (post_eps, norm_eps, None if h is None else h.dtype, x.dtype, geo, x.shape, direct, r is not None,
                   None if norm is None else norm_b.shape, None if norm is None else norm_b.dtype)
        return r if y is None else y if r is None else (r, y)

    @staticmethod
    def backward(ctx, *gos):
        base, h, res_scale, gate, post_w, post_b, norm_w, stats = ctx.saved_tensors
        post_eps, norm_eps, h_dtype, x_dtype, geo, shape, direct, has_r, nb_shape, nb_dtype = ctx.cfg
        gr = gos[0] if has_r else None
        gy = gos[-1] if norm_w is not None else None
        need = ctx.needs_input_grad[:8]
        if gr is None and gy is None:
            return (None,) * 11
        of_copy = gr is not None and h_dtype is None  # from a differentiated backward alone
        if of_copy or torch.is_grad_enabled() or _dispatch_modes() or _pre_dispatch() or not (
                _in_memory(gr) and _in_memory(gy)):
            post = None if post_w is None else (post_w, post_b, post_eps)
            return _residual_norm_backward_composite(base, h, res_scale, gate, post, norm_w, nb_shape, nb_dtype, norm_eps, gr,
                                                     gy, h_dtype, x_dtype, need) + (None, None, None)
        # a saved-tensor hook may have given any of them other strides
        base, h, res_scale, gate, post_w, post_b, norm_w, stats = map(
            _contiguous, (base, h, res_scale, gate, post_w, post_b, norm_w, stats))
        got = _residual_norm_backward(gr, gy, base, h, stats, norm_w, nb_shape, res_scale, gate, post_w, post_b, geo, shape,
                                      x_dtype, h_dtype, need, direct)
        if direct:  # float32 parameters, as their gradients
            return got + (None, None, None)
        gx, gh, gs, gg, *gp, gb = got
        like = lambda g, t: g if g is None or t.dtype is torch.float32 else g.to(t.dtype)  # noqa: E731
        return (gx, gh, like(gs, res_scale), gg, *map(like, gp, (post_w, post_b, norm_w)), None if gb is None else
                gb.to(nb_dtype), None, None, None)


def _residual_norm_backward_composite(base, h, res_scale, gate, post, norm_w, nb_shape, nb_dtype, norm_eps, gr, gy, h_dtype,
                                      x_dtype, need):
    """The same gradients from their formulas in differentiable torch operations."""
    ref = next(t for t in (base, h, gr, gy) if t is not None)
    cf = (1, -1) + (1,) * (ref.dim() - 2)
    pixels = [d for d in range(ref.dim()) if d != 1]

    def like(g, t):
        return g.reshape(t.shape).to(t.dtype)

    dr = None if gr is None else gr.float()
    gnw = gnb = None
    if gy is not None:
        r = base.float()
        if x_dtype != torch.float32 and h is not None:
            r = r + composite.residual_branch(h, res_scale, gate, post)  # base is x
        hat, rho = composite.standardised(r, norm_eps)
        gy = gy.float()
        d = composite.standardised_grad(gy * norm_w.float().view(cf), hat, rho)
        dr = d if dr is None else dr + d
        gnw = like((gy * hat).sum(pixels), norm_w) if need[6] else None
        gnb = gy.sum(pixels).reshape(nb_shape).to(nb_dtype) if need[7] else None
    gx = dr.to(x_dtype) if need[0] else None
    gh = gs = gg = gpw = gpb = None
    if h is None:
        gh = dr.to(h_dtype) if h_dtype is not None and need[1] else None
        return gx, gh, gs, gg, gpw, gpb, gnw, gnb
    n = h.float()
    if post is not None:
        phat, prho = composite.standardised(n, post[2])
        n = phat * post[0].float().view(cf) + post[1].float().view(cf)
    g = None
    if gate is not None:
        g = (gate if gate.shape == h.shape else gate.reshape(gate.shape[:2] + (1,) * (h.dim() - 2))).float()
    u = n if g is None else n * g
    du = dr
    if res_scale is not None:
        gs = like((dr * u).sum(pixels), res_scale) if need[2] else None
        du = dr * res_scale.float().view(cf)
    dn = du
    if gate is not None:
        if need[3]:
            gg = du * n
            if gate.shape != h.shape:
                gg = gg.flatten(2).sum(2)
            gg = like(gg, gate)
        dn = du * g
    if post is not None:
        gpw = like((dn * phat).sum(pixels), post[0]) if need[4] else None
        gpb = like(dn.sum(pixels), post[1]) if need[5] else None
        dn = composite.standardised_grad(dn * post[0].float().view(cf), phat, prho)
    gh = dn.to(h_dtype) if need[1] else None
    return gx, gh, gs, gg, gpw, gpb, gnw, gnb


def residual_norm_train(x, h, norm=None, res_scale=None, gate=None, post=None):
    """Differentiable residual_norm on the HIP kernels (forward and backward): (r, y)."""
    if h is None:
        raise RuntimeError("residual_norm needs a branch")
    pw, pb, pe = post or (None, None, 0.0)
    nw, nb, ne = norm or (None, None, 0.0)
    out = ResidualNormFunction.apply(_contiguous(x), _contiguous(h), res_scale, _contiguous(gate), pw, pb, nw, nb, pe, ne)
    return (out, None) if norm is None else out


def layernorm_cf_train(x, weight, bias, eps, copy=False):
    """Differentiable layernorm_cf on the HIP kernels (forward and backward).  copy: the backward reads a copy of x that the
    forward makes, so that x may be changed in place after it."""
    if not copy:
        return ResidualNormFunction.apply(_contiguous(x), None, None, None, None, None, weight, bias, 0.0, eps)
    # the copy is an output, which a differentiated backward reaches x through
    return ResidualNormFunction.apply(_contiguous(x), None, None, None, None, None, weight, bias, 0.0, eps, True)[1]


def _grad_list(ts):
    """What the library takes of a list of gradients: device index, types, sizes and addresses.  (A model has hundreds:
    the loops run in C.)"""
    index = ts[0].get_device()
    if index < 0 or set(map(torch.Tensor.get_device, ts)) != {index}:
        raise RuntimeError("gradients must be on one HIP device")
    try:
        types = array("i", map(_lib.TYPES.__getitem__, map(_DTYPE, ts)))
    except KeyError as e:
        raise RuntimeError(f"gradients must be float32, bfloat16 or float16, got {e.args[0]}") from None
    return index, types, array("q", map(torch.Tensor.numel, ts)), array("Q", map(torch.Tensor.data_ptr, ts))


_DTYPE = operator.attrgetter("dtype")


def _norm_kind(norm_type):
    kind = {2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}.get(float(norm_type))
    if kind is None:
        raise RuntimeError("norm_type must be 2 or inf")
    return kind


def _all_contiguous(ts):
    if all(map(torch.Tensor.is_contiguous, ts)):
        return ts
    with torch.no_grad():
        return [t.contiguous() for t in ts]


def _as_stored(keep, grads, out, sizes, src):
    """Puts into src the addresses of copies (held in `keep`) of gradients whose memory has the other sign than their
    output's: views of an imaginary part, of which only those of one element are contiguous."""
    i = -1
    for _ in range(sizes.count(1)):
        i = sizes.index(1, i + 1)
        g, o = grads[i], out[i]
        if g.is_neg() != o.is_neg():
            with torch.no_grad():
                keep.append(-g if o.is_neg() else g.resolve_neg())
            src[i] = keep[-1].data_ptr()


def _clip(grads, out, max_norm, norm_type):
    """The norm of contiguous grads, and (out not None) their clipped values into contiguous out."""
    _untraced("grad_norm" if out is None else "clip_grads")
    kind = _norm_kind(norm_type)
    max_norm = 0.0 if out is None else float(max_norm)
    if not max_norm >= 0.0:
        raise RuntimeError("max_norm must be at least 0")
    if not grads:
        return torch.tensor(0.0)
    lib = _lib.load()
    index, types, sizes, src = _grad_list(grads)
    dst = src
    keep = []
    if out is not None and out is not grads:
        oi, ot, on, dst = _grad_list(out)
        if oi != index or ot != types or on != sizes:
            raise RuntimeError("out must have the gradients' sizes and types, on their device")
        _as_stored(keep, grads, out, sizes, src)
    n = len(grads)
    dev = grads[0].device
    tables = (src, dst, sizes, types)  # held until the library has read them
    src_at, dst_at, sizes_at, types_at = (a.buffer_info()[0] for a in tables)
    nbytes = lib.cvn_grad_norm_workspace(sizes_at, n)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    st = _stream(dev)
    ws = _scratch(dev, st)
    with _on(dev), ws.lock:
        if out is None:
            rc = lib.cvn_grad_norm(src_at, sizes_at, types_at, n, kind, norm.data_ptr(), ws.ptr(nbytes), nbytes, st)
        else:
            rc = lib.cvn_clip_grads(src_at, dst_at, sizes_at, types_at, n, kind, max_norm, norm.data_ptr(),
                                    ws.ptr(nbytes), nbytes, st)
    del tables, keep
    _lib.check(rc, "grad_norm" if out is None else "clip_grads")
    return norm


def _tensors(ts):
    return [ts] if isinstance(ts, torch.Tensor) else list(ts)


def grad_norm(grads, norm_type=2.0):
    """The norm over all elements of many tensors (2, or math.inf for the largest magnitude): a float32 scalar on their
    device, accumulated in 64 bits.  grads: tensors of any shapes, float32, bfloat16 or float16, on one device.  (Not
    differentiable; no host wait.)"""
    return _clip(_all_contiguous(_tensors(grads)), None, None, norm_type)


def _written(ts):
    """The library wrote these tensors: autograd sees it as it sees torch's in-place operations.  (Inference tensors have
    no version, and are passed over.)"""
    torch.autograd.graph.increment_version(ts)


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """(grads scaled by min(1, max_norm / (norm + 1e-6)), norm).  The scaled gradients go to new tensors, or to `out`:
    contiguous tensors of the same types and sizes, each its own gradient or memory apart from all others."""
    grads = _tensors(grads)
    if out is None:
        out = [torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in grads]
    else:
        out = _tensors(out)
        if len(out) != len(grads):
            raise RuntimeError("out must hold a tensor for each gradient")
        if not all(map(torch.Tensor.is_contiguous, out)):
            raise RuntimeError("out must be contiguous")
    norm = _clip(_all_contiguous(grads), out, max_norm, norm_type)
    _written(out)
    return out, norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scales the parameters' .grad in place so that their norm is at most max_norm; returns the norm they had, in float32.
    As torch.nn.utils.clip_grad_norm_, for gradients that are float32, bfloat16 or float16 on one HIP device, each in memory
    of its own (a parameter that is passed twice is refused), max_norm >= 0 and norm_type 2 or math.inf; RuntimeError
    otherwise.  error_if_nonfinite waits for the norm and raises before any gradient changes.  Strided gradients are copied
    there and back."""
    grads = [g for g in [p.grad for p in _tensors(parameters)] if g is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of the gradients is {norm.item()}")
    dense = _all_contiguous(grads)
    if dense is not grads:
        for g in grads:
            if 0 in g.stride() and any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
                raise RuntimeError("a gradient's elements share memory")
        strided = [g for g, d in zip(grads, dense) if d is not g and g.numel()]
        if len({(g.data_ptr(), g.shape, g.stride()) for g in strided}) != len(strided):
            raise RuntimeError("two gradients share memory")
    norm = _clip(dense, dense, max_norm, norm_type)
    if dense is not grads:
        with torch.no_grad():
            for g, d in zip(grads, dense):
                if d is not g:
                    g.copy_(d)
        dense = [d for g, d in zip(grads, dense) if d is g]
    _written(dense)
    return norm


class MXFP4(NamedTuple):
    """A map (B,C,*) or matrix (N,C) in microscaled 4-bit floating point: its channels in blocks of 32, each a scale
    2^(s - 127) and 32 codes of a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6, stored by pixels.  codes (B,*,16 blocks) and
    scales (B,*,blocks) are uint8, a byte of codes holds the even channel in its lower half; channels is C."""
    codes: torch.Tensor
    scales: torch.Tensor
    channels: int

    @property
    def shape(self):
        return (self.codes.shape[0], self.channels, *self.codes.shape[1:-1])


def _values(t):
    """A contiguous tensor of t's values as stored (None for None): a view of an imaginary part may hold their negatives."""
    if t is None:
        return None
    t = t if t.is_contiguous() else t.contiguous()
    if t.is_neg():
        t = t.resolve_neg()
    if not t.data_ptr() and t.numel():  # (the library would take it for none)
        raise RuntimeError("a tensor that stands for others has no memory to compute on")
    return t


def _mx_parts(q, what):
    """((B, C, pixels), codes, scales) of an MXFP4 argument, contiguous and aligned."""
    codes, scales, C = q
    blocks = (int(C) + 31) // 32
    if not (isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor)) or codes.dtype is not torch.uint8 \
            or scales.dtype is not torch.uint8 or C < 1 or codes.dim() < 2 or codes.shape[:-1] != scales.shape[:-1] \
            or codes.shape[-1] != 16 * blocks or scales.shape[-1] != blocks:
        raise RuntimeError(f"{what}: codes (B,*,16 blocks) and scales (B,*,blocks) must be uint8 of {blocks} blocks")
    if codes.get_device() < 0 or scales.get_device() != codes.get_device():
        raise RuntimeError(f"{what} must be on one HIP device")
    codes, scales = _contiguous(codes), _contiguous(scales)
    if codes.data_ptr() % 16:
        codes = codes.clone()
    return (codes.shape[0], int(C), math.prod(codes.shape[1:-1])), codes, scales


def _mx_map(x, what):
    """(B, C, pixels) of a map to be quantised."""
    if x.get_device() < 0 or x.dtype not in _lib.TYPES:
        raise RuntimeError(f"{what} needs a float32, bfloat16 or float16 tensor on a HIP device")
    if x.dim() < 2 or x.shape[1] < 1:
        raise RuntimeError(f"{what} needs (B,C,*) with channels")
    return x.shape[0], x.shape[1], math.prod(x.shape[2:])


def _mx_empty(x, C):
    """The memory of x's MXFP4 form."""
    lead = (x.shape[0], *x.shape[2:])
    blocks = (C + 31) // 32
    return (torch.empty((*lead, 16 * blocks), dtype=torch.uint8, device=x.device),
            torch.empty((*lead, blocks), dtype=torch.uint8, device=x.device))


def quantize_mxfp4(x):
    """A map (B,C,*) or matrix (N,C) in MXFP4: blocks of 32 channels with the scale 2^(floor(log2 max|x|) - 2) and each
    value the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it, ties to the even code, at most 6 (2^-127 is the smallest
    scale).  A block with an infinity or a NaN becomes NaN.  x: float32, bfloat16 or float16."""
    _untraced("quantize_mxfp4")
    B, C, HW = _mx_map(x, "quantize_mxfp4")
    lib = _lib.load()
    x = _values(x)
    codes, scales = _mx_empty(x, C)
    with _on(x.device):
        rc = lib.cvn_mxfp4_quantize(x.data_ptr(), _lib.TYPES[x.dtype], B, C, HW, codes.data_ptr(), scales.data_ptr(),
                                    _stream(x.device))
    _lib.check(rc, "quantize_mxfp4")
    return MXFP4(codes, scales, C)


def dequantize_mxfp4(q, dtype=torch.float32):
    """The values of an MXFP4 map or matrix as a tensor (B,C,*)."""
    _untraced("dequantize_mxfp4")
    (B, C, HW), codes, scales = _mx_parts(q, "dequantize_mxfp4")
    if dtype not in _lib.TYPES:
        raise RuntimeError("dequantize_mxfp4 gives float32, bfloat16 or float16")
    lib = _lib.load()
    dev = codes.device
    y = torch.empty((B, C, *codes.shape[1:-1]), dtype=dtype, device=dev)
    with _on(dev):
        rc = lib.cvn_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), B, C, HW, y.data_ptr(), _lib.TYPES[dtype],
                                      _stream(dev))
    _lib.check(rc, "dequantize_mxfp4")
    return y


def _mx_weight(weight, C, index):
    """(N, C) of a float matrix to be quantised."""
    if weight.get_device() != index or weight.dim() < 2 or math.prod(weight.shape[2:]) != 1 or weight.dtype not in _lib.TYPES:
        raise RuntimeError("weight must be a matrix (N,C) or (N,C,1,1) on the device of x: float32, bfloat16 or float16")
    if weight.shape[1] != C or weight.shape[0] < 1:
        raise RuntimeError("weight does not match input channels")
    return weight.shape[0]


def conv1x1_mxfp4(x, weight, bias=None, act=None, residual=None, res_scale=None, out=None, dtype=None):
    """conv1x1 of MXFP4 operands: act(W x + b) [then res_scale * . + residual], the products of 4-bit values summed in
    float32 and the result rounded once.

    x: a map (B,C,*) of float32, bfloat16 or float16, quantised in the call, or an MXFP4 one; weight: an MXFP4 matrix, or a
    float (N,C) or (N,C,1,1), quantised in the call.  The result has x's type (of an MXFP4 x the residual's, or dtype).
    residual and out have the result's shape and type, and may be one tensor.  Forward only; for gradients see
    conv1x1_mxfp4_train."""
    _untraced("conv1x1_mxfp4")
    lib = _lib.load()
    if act not in (None, "gelu"):
        raise RuntimeError(f"unknown activation {act!r}")
    xc = xs = wc = ws = None
    if isinstance(x, MXFP4):
        (B, C, HW), xc, xs = _mx_parts(x, "x")
        x, dev, space = None, xc.device, xc.shape[1:-1]
        dtype = dtype or (torch.float32 if residual is None else residual.dtype)
        if dtype not in _lib.TYPES:
            raise RuntimeError("conv1x1_mxfp4 gives float32, bfloat16 or float16")
    else:
        B, C, HW = _mx_map(x, "conv1x1_mxfp4")
        if dtype not in (None, x.dtype):
            raise RuntimeError("the result has the type of x")
        x = _values(x)
        dev, space, dtype = x.device, x.shape[2:], x.dtype
    index = dev.index
    if isinstance(weight, MXFP4):
        (N, wC, one), wc, ws = _mx_parts(weight, "weight")
        weight = None
        if wC != C or one != 1 or N < 1 or wc.get_device() != index:
            raise RuntimeError("weight does not match input channels")
    else:
        N = _mx_weight(weight, C, index)
        weight = _values(weight)
    shape = (B, N, *space)
    for t, what in ((residual, "residual"), (out, "out")):
        if t is not None and (tuple(t.shape) != shape or t.dtype is not dtype or t.get_device() != index):
            raise RuntimeError(f"{what} must have the result's shape and type")
    if out is not None and (not out.is_contiguous() or out.is_neg()):
        raise RuntimeError("out must be contiguous, and no negated view")
    keep = []
    b, s = _param32(keep, bias, N, index, "bias"), _param32(keep, res_scale, N, index, "res_scale")
    residual = _values(residual)
    y = torch.empty(shape, dtype=dtype, device=dev) if out is None else out
    nbytes = 0 if x is None and weight is None else lib.cvn_conv1x1_mxfp4_workspace(x is None, weight is None, B, C, HW, N)
    st = _stream(dev)
    work = _scratch(dev, st)
    with _on(dev), work.lock:
        rc = lib.cvn_conv1x1_mxfp4(_ptr(x), _ptr(xc), _ptr(xs), B, C, HW, _ptr(weight),
                                   0 if weight is None else _lib.TYPES[weight.dtype], _ptr(wc), _ptr(ws), N, b,
                                   _lib.ACT_GELU if act else _lib.ACT_NONE, _ptr(residual), s, y.data_ptr(),
                                   _lib.TYPES[dtype], work.ptr(nbytes), nbytes, st)
    _lib.check(rc, "conv1x1_mxfp4")
    if out is not None:
        _written([out])
    return y


def conv1x1_mxfp4_backward(grad_y, x, weight, need=(True, True, True)):
    """Gradients of conv1x1_mxfp4's product and bias, straight through the quantisation: (x, weight, bias), None where
    not asked for by `need`.  grad_y (B,N,*): float32, bfloat16 or float16, the type of x's gradient; the others are float32,
    weight's (N,C).  (Parts of an operand below 2^-126 count as zeros.)  x, weight: the MXFP4 operands of the forward (x
    None without weight's gradient, weight None without x's, where the other gives the channels)."""
    _untraced("conv1x1_mxfp4_backward")
    B, N, HW = _mx_map(grad_y, "conv1x1_mxfp4_backward")
    nx, nw, nb = need
    if (nx and weight is None) or (nw and x is None):
        raise RuntimeError("conv1x1_mxfp4_backward needs the operand")
    index = grad_y.get_device()
    C, xc, xs, wc, ws = 1, None, None, None, None
    if x is not None and nw:
        (xB, C, xHW), xc, xs = _mx_parts(x, "x")
        if xB != B or xc.shape[1:-1] != grad_y.shape[2:] or xc.get_device() != index:
            raise RuntimeError("x does not match the gradient")
    if weight is not None and nx:
        (wN, wC, one), wc, ws = _mx_parts(weight, "weight")
        if wN != N or one != 1 or (xc is not None and wC != C) or wc.get_device() != index:
            raise RuntimeError("weight does not match the gradient")
        C = wC
    gy = _values(grad_y)
    dev = gy.device
    gx = torch.empty((B, C, *gy.shape[2:]), dtype=gy.dtype, device=dev) if nx else None
    gw = torch.empty((N, C), dtype=torch.float32, device=dev) if nw else None
    gb = torch.empty((N,), dtype=torch.float32, device=dev) if nb else None
    _mx_grads(gy, _ptr(xc), _ptr(xs), _ptr(wc), _ptr(ws), B, C, HW, N, gx, gw, gb)
    return gx, gw, gb


@functools.lru_cache(maxsize=1024)
def _mx_grad_workspace(B, C, HW, N):
    """Bytes of scratch of a gradient of the matrix (the library's answer depends on nothing else)."""
    return _lib.load().cvn_conv1x1_mxfp4_bwd_workspace(B, C, HW, N)


def _mx_grads(gy, xc, xs, wc, ws, B, C, HW, N, gx, gw, gb):
    """The launches behind conv1x1_mxfp4's gradients."""
    lib = _lib.load()
    dev = gy.device
    nbytes = _mx_grad_workspace(B, C, HW, N) if gw is not None else 0
    st = _stream(dev)
    work = _scratch(dev, st)
    with _on(dev), work.lock:
        rc = lib.cvn_conv1x1_mxfp4_bwd(gy.data_ptr(), _lib.TYPES[gy.dtype], xc, xs, wc, ws, B, C, HW, N, _ptr(gx), _ptr(gw),
                                       _ptr(gb), work.ptr(nbytes), nbytes, st)
    _lib.check(rc, "conv1x1_mxfp4_backward")


@functools.lru_cache(maxsize=1024)
def _mx_layout(rows, C, N, keep_x, keep_w):
    """Where a forward keeps its operands in one buffer: (codes and scales of x, of the matrix, bytes), None for what is
    not kept."""
    blocks = (C + 31) // 32
    at, out = 0, []
    for n, wanted in ((16 * rows, keep_x), (16 * N, keep_w), (rows, keep_x), (N, keep_w)):
        out.append(at if wanted else None)
        at += (n * blocks + 255) // 256 * 256 if wanted else 0
    return out[0], out[2], out[1], out[3], at


class Conv1x1MXFP4Function(torch.autograd.Function):
    """conv1x1_mxfp4 of a float map and matrix, with gradients straight through both quantisations.  Keeps the operands that
    the gradients need in MXFP4, 17/128 of float32's bytes, in one buffer."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        if _dispatch_modes() or _function_modes() or _tracing_state() is not None:
            _untraced("conv1x1_mxfp4_train")
        lib = _lib.load()
        B, C, HW = _mx_map(x, "conv1x1_mxfp4_train")
        dev, dtype = x.device, x.dtype
        index = dev.index
        N = _mx_weight(weight, C, index)
        x, w = _values(x), _values(weight)
        keep = []
        b = _param32(keep, bias, N, index, "bias")
        nx, nw = ctx.needs_input_grad[:2]
        where = _mx_layout(B * HW, C, N, nw, nx)
        kept = torch.empty(where[4], dtype=torch.uint8, device=dev) if nx or nw else None
        base = 0 if kept is None else kept.data_ptr()
        xc, xs, wc, ws = (None if o is None or not base else base + o for o in where[:4])
        y = torch.empty((B, N, *x.shape[2:]), dtype=dtype, device=dev)
        nbytes = 0 if nx and nw else lib.cvn_conv1x1_mxfp4_workspace(xc is not None, wc is not None, B, C, HW, N)
        st = _stream(dev)
        work = _scratch(dev, st)
        with _on(dev), work.lock:
            rc = lib.cvn_conv1x1_mxfp4(x.data_ptr(), xc, xs, B, C, HW, w.data_ptr(), _lib.TYPES[w.dtype], wc, ws, N, b, 0, None,
                                       None, y.data_ptr(), _lib.TYPES[dtype], work.ptr(nbytes), nbytes, st)
        _lib.check(rc, "conv1x1_mxfp4_train")
        ctx.save_for_backward(kept)
        ctx.cfg = (where, x.shape, weight.shape, weight.dtype, None if bias is None else (bias.shape, bias.dtype))
        return y

    @staticmethod
    def backward(ctx, gy):
        # (a backward that is itself to be differentiated gives gradients that refuse it)
        return _mx_backward_once(ctx, gy) if torch.is_grad_enabled() else _mx_backward(ctx, gy)


def _mx_backward(ctx, gy):
    kept, = ctx.saved_tensors
    where, x_shape, w_shape, w_dtype, bias = ctx.cfg
    nx, nw, nb = ctx.needs_input_grad
    if not _in_memory(gy) or not _in_memory(kept):
        raise RuntimeError("conv1x1_mxfp4's gradients are of plain tensors")
    gy, kept = _values(gy), _contiguous(kept)
    dev = gy.device
    if kept is not None and (kept.device != dev or kept.dtype is not torch.uint8 or kept.numel() != where[4]):
        raise RuntimeError("a hook has changed what conv1x1_mxfp4_train kept")
    B, C, N, HW = x_shape[0], x_shape[1], w_shape[0], math.prod(x_shape[2:])
    base = 0 if kept is None else kept.data_ptr()
    if base % 16:  # (a saved-tensor hook may have moved it)
        kept = kept.clone()
        base = kept.data_ptr()
    xc, xs, wc, ws = (None if o is None or not base else base + o for o in where[:4])
    gx = torch.empty(x_shape, dtype=gy.dtype, device=dev) if nx else None
    gw = torch.empty(w_shape, dtype=torch.float32, device=dev) if nw else None
    gb = torch.empty(bias[0], dtype=torch.float32, device=dev) if nb else None
    _mx_grads(gy, xc, xs, wc, ws, B, C, HW, N, gx, gw, gb)
    if nw and w_dtype is not torch.float32:
        gw = gw.to(w_dtype)
    if nb and bias[1] is not torch.float32:
        gb = gb.to(bias[1])
    return gx, gw, gb


_mx_backward_once = torch.autograd.function.once_differentiable(_mx_backward)


_RECORDING = "conversenet_amd.recording"


def _accumulator(leaf):
    """The node that a leaf's gradients end in: the one that lives, or a new one."""
    return leaf.view_as(leaf).grad_fn.next_functions[0][0]


def _recorded_too(device, stream_id):
    """Whether a stream is part of a recording (one that forks onto it); the null stream cannot be."""
    if stream_id == 0:
        return False
    with torch.cuda.stream(torch.cuda.Stream(stream_id=stream_id, device_index=device, device_type=_DEVICE_TYPE)):
        return torch._C._cuda_isCurrentStreamCapturing()


_DEVICE_TYPE = 1  # (torch's number for devices named cuda)


def _elsewhere(t):
    """Whether a node that a tensor's gradient reaches was made on a stream outside of the recording on the current one."""
    return not all(_recorded_too(*s) for s in _lib.graph_streams(t))


def _own_leaves(leaves, stream):
    """Refuses a recording whose leaves are part of a graph from outside of it: such a leaf's node lives on the stream that it
    was made on, the recorded backward would make that stream wait for the recording, and the recording's end would end the
    process.  (A mark says that a recording on the stream has the leaf's node.)"""
    if any(_accumulator(t).metadata.get(_RECORDING) != stream and _elsewhere(t) for t in leaves):
        raise RuntimeError("a training pass cannot be recorded while a graph made before holds one of its leaves: let go of "
                           "that graph's outputs first")


def _own_operands(operands, stream):
    """Refuses a recording whose operands come from nodes outside of it, leaves or not (see _own_leaves)."""
    _own_leaves([t for t in operands if t.is_leaf], stream)
    if any(not t.is_leaf and _elsewhere(t) for t in operands):
        raise RuntimeError("a training pass cannot be recorded with an operand whose graph, or a leaf of it, was made outside of the "
                           "recording: let go of earlier graphs' outputs first, and make views in the recording")


def conv1x1_mxfp4_train(x, weight, bias=None):
    """Differentiable conv1x1_mxfp4 of a float map (B,C,*) and matrix (N,C) or (N,C,1,1), both quantised in the call: the
    gradients pass the quantisation unchanged, those of x and weight are products with the other's 4-bit values.  (Not
    differentiable twice.  Recorded into a graph, nothing that its gradients reach is in a graph that lives from before.)"""
    if isinstance(x, MXFP4) or isinstance(weight, MXFP4):
        raise RuntimeError("conv1x1_mxfp4_train quantises x and weight itself")
    if x.is_cuda and torch.is_grad_enabled() and _capturing(stream := _stream(x.device)):
        operands = [t for t in (x, weight, bias) if t is not None and t.requires_grad]
        _own_operands(operands, stream)
        y = Conv1x1MXFP4Function.apply(x, weight, bias)
        for t in operands:
            if t.is_leaf:
                _accumulator(t).metadata[_RECORDING] = stream
        return y
    return Conv1x1MXFP4Function.apply(x, weight, bias)


def copy_(dst, src):
    """Plain device copy through the library (HBM calibration kernel)."""
    lib = _lib.load()
    _need_hip(dst, src)
    _lib.check(lib.cvn_copy_f32(src.data_ptr(), dst.data_ptr(), src.numel(), _stream(src.device)), "copy")
    return dst
