"""Glue between torch tensors and the C ABI: enum codes, pointer extraction, status checks."""
import contextlib
import ctypes
import os

import torch

from ... import _clib

PT_BF16, PT_F16, PT_F32 = 0, 1, 2
PT_E4M3, PT_E5M2, PT_E2M1 = 0, 1, 2
PT_TENSORWISE, PT_ROWWISE, PT_BLOCKWISE, PT_MX_BLOCKWISE = 0, 1, 2, 3
PT_MX_ROW, PT_MX_COL, PT_MX_ROW_2D, PT_MX_COL_2D, PT_MX_ROW_RHT, PT_MX_COL_RHT = 1, 2, 4, 8, 16, 32
PT_MX_ROW_SR, PT_MX_COL_SR = 64, 128
PT_ERR_INVALID = -1

_SRC = {torch.bfloat16: PT_BF16, torch.float16: PT_F16, torch.float32: PT_F32}
_FMT = {torch.float8_e4m3fn: PT_E4M3, torch.float8_e5m2: PT_E5M2, torch.float4_e2m1fn_x2: PT_E2M1}


check = _clib.check


def lib():
    return _clib.load()


def src_code(dtype) -> int:
    try:
        return _SRC[dtype]
    except KeyError:
        raise TypeError(f"unsupported high-precision dtype {dtype}") from None


def fmt_code(dtype) -> int:
    try:
        return _FMT[dtype]
    except KeyError:
        raise TypeError(f"unsupported quantized dtype {dtype}") from None


def ptr(t):
    return None if t is None else t.data_ptr()      # a plain int: ctypes converts it by the argument's type


def stream(device=None):
    idx = None if device is None else device.index
    # the handle alone: building a torch Stream object around it costs as much as a launch
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if idx is None else idx)


_NO_GUARD = contextlib.nullcontext()


def on_device(device):
    """Context in which `device` is the current CUDA device; free when it already is (the usual case: one process
    per GPU), a torch device guard otherwise."""
    idx = device.index
    if idx is None or idx == torch._C._cuda_getDevice():
        return _NO_GUARD
    return torch.cuda.device(device)


def require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("primus_turbo (B200) operators take CUDA tensors only; there is no CPU path")


_status = {}
_poll = {}
_host_status = {}


def status_word(device) -> torch.Tensor:
    """Per-device int32 the kernels write PT_ERR_TIMEOUT into if one of their bounded waits gives up.  The GEMM entry
    points get it as their `status` argument; it is also registered with the library as the word the quantizers (which
    have no such argument) report into."""
    idx = torch.device(device).index
    if idx is None:
        idx = torch.cuda.current_device()
    if idx not in _status:
        _status[idx] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{idx}")
        with torch.cuda.device(idx):
            check(lib().pt_set_default_status(ptr(_status[idx])), "set_default_status")
    return _status[idx]


def mapped_status(device):
    """Address of the device's status word in pinned host memory, which the kernels of gemm_bias_act, qk_norm_rope and
    moe_few_tokens write directly (mapped, so the address is the device's too).  Raises if a kernel launched earlier has reported
    an error into it: nothing is waited for, the error of a launch surfaces at a following call, at check_status(), or with
    PT_CHECK_STATUS=1 at the launch itself (launched()).  One host load: a copy and an event per call, as poll_status makes, would cost
    an operator on one token as much as its kernel."""
    w = _host_status.get(device.index)
    if w is None:
        t = torch.zeros(1, dtype=torch.int32).pin_memory()
        w = _host_status[device.index] = (t, ctypes.c_int32.from_address(t.data_ptr()), t.data_ptr())
    if w[1].value != 0:
        code, w[1].value = w[1].value, 0
        _raise(code)
    return w[2]


# os.environ's own table: a look-up through os.environ takes 0.8 us, a twentieth of a whole call on one token
_environ = getattr(os.environ, "_data", os.environb)


def launched(device):
    """After a launch that was given mapped_status: the synchronising check of PT_CHECK_STATUS=1, as poll_status makes it."""
    if _environ.get(b"PT_CHECK_STATUS") == b"1" and not torch.cuda.is_current_stream_capturing():
        check_status(device)


def _raise(code):
    if code == PT_ERR_INVALID:
        raise RuntimeError("a kernel was given an index outside of its table (a position beyond the cos / sin rows); the rows of that "
                           "launch with such an index are zeros")
    raise RuntimeError(f"a kernel gave up waiting on a barrier (status {code}); the output of that launch is invalid")


def check_status(device):
    """Synchronises and raises if a kernel reported an expired wait or an index outside of its table since the last check."""
    s = status_word(device)
    code = int(s.item())
    if code != 0:
        s.zero_()
        _raise(code)
    mapped_status(s.device)


def poll_status(device):
    """Called by the GEMM wrappers after a launch.  PT_CHECK_STATUS=1: a synchronising check_status().  Otherwise a check
    that never waits for the device: the status word is copied to pinned host memory asynchronously, at most one copy in
    flight; a later call that finds the copy complete reads it and raises if a kernel had given up.  An error therefore
    surfaces at a following operator call (or at an explicit check_status()), not at the launch that caused it."""
    if os.environ.get("PT_CHECK_STATUS") == "1":
        if not torch.cuda.is_current_stream_capturing():
            check_status(device)
        return
    idx = torch.device(device).index
    if idx is None:
        idx = torch.cuda.current_device()
    p = _poll.get(idx)
    if p is None:
        p = _poll[idx] = {"host": torch.zeros(1, dtype=torch.int32).pin_memory(), "event": torch.cuda.Event(), "pending": False}
    if torch.cuda.is_current_stream_capturing():
        return
    if p["pending"]:
        if not p["event"].query():
            return
        p["pending"] = False
        code = int(p["host"][0])
        if code != 0:
            status_word(device).zero_()
            _raise(code)
    p["host"].copy_(status_word(device), non_blocking=True)
    p["event"].record(torch.cuda.current_stream(idx))
    p["pending"] = True


