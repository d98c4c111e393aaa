"""ctypes binding of libq35b200.so: tensors are bound BY NAME, as the reference's hosts bind kernel IO
(tools/board/axrun.cc:55-110; models/qwen35_2b/whole/src/q35_layer_mc.py:915-916).

There is no fallback: if the shared library is missing or a call fails, an exception is raised.
"""
import ctypes
import json
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libq35b200.so")
MAX_DIMS = 6

# AX engine element codes of the reference's IO tables (tools/manifest/onnx_io.py:21-32)
U8, F32, I32, BF16, F16, E4M3, FP4 = 1, 3, 6, 9, 10, 11, 15
_DTYPE_CODE = {
    torch.uint8: U8, torch.float32: F32, torch.int32: I32, torch.bfloat16: BF16, torch.float16: F16,
    torch.float8_e4m3fn: E4M3, torch.int8: U8,  # int8 KV rows travel as bytes (the AX table has no int8 code)
}
for _n, _c in (("float8_e8m0fnu", U8), ("float4_e2m1fn_x2", U8)):  # scale / packed-FP4 views are raw bytes
    if hasattr(torch, _n):
        _DTYPE_CODE[getattr(torch, _n)] = _c


class Q35Error(RuntimeError):
    def __init__(self, status, text):
        super().__init__(f"q35b200 status {status}: {text}")
        self.status = status


class _IO(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("ptr", ctypes.c_void_p), ("bytes", ctypes.c_size_t),
                ("dtype", ctypes.c_int), ("ndim", ctypes.c_int), ("shape", ctypes.c_int64 * MAX_DIMS)]


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise Q35Error(-1, f"{LIB_PATH} is missing: build it with `python -m ax_dsl_kernels_b200.build` "
                               "(there is no CPU or PyTorch fallback)")
        L = ctypes.CDLL(LIB_PATH)
        L.q35_run.argtypes = [ctypes.c_char_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
        L.q35_run.restype = ctypes.c_int
        L.q35_workspace_bytes.argtypes = [ctypes.c_char_p, ctypes.POINTER(_IO), ctypes.c_int]
        L.q35_workspace_bytes.restype = ctypes.c_int64
        L.q35_io_table.argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_size_t]
        L.q35_io_table.restype = ctypes.c_int
        L.q35_role_count.restype = ctypes.c_int
        L.q35_role_name.argtypes = [ctypes.c_int]
        L.q35_role_name.restype = ctypes.c_char_p
        L.q35_last_error.restype = ctypes.c_char_p
        L.q35_device_status.argtypes = [ctypes.c_void_p]
        L.q35_device_status.restype = ctypes.c_int
        L.q35_version.restype = ctypes.c_int
        L.q35_launch_count.restype = ctypes.c_longlong
        _lib = L
    return _lib


def _table(tensors):
    arr = (_IO * len(tensors))()
    keep = []
    for i, (name, t) in enumerate(tensors.items()):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: tensor must be contiguous")
        if t.dim() > MAX_DIMS:
            raise ValueError(f"{name}: more than {MAX_DIMS} dims")
        code = _DTYPE_CODE.get(t.dtype)
        if code is None:
            raise TypeError(f"{name}: unsupported dtype {t.dtype}")
        b = name.encode()
        keep.append(b)
        arr[i].name = b
        arr[i].ptr = t.data_ptr()
        arr[i].bytes = t.numel() * t.element_size()
        arr[i].dtype = code
        arr[i].ndim = t.dim()
        for d in range(t.dim()):
            arr[i].shape[d] = t.shape[d]
    return arr, keep


def _check(st):
    if st != 0:
        raise Q35Error(st, lib().q35_last_error().decode())


def workspace_bytes(role, **tensors):
    arr, _keep = _table(tensors)
    n = lib().q35_workspace_bytes(role.encode(), arr, len(tensors))
    if n < 0:
        raise Q35Error(-n, lib().q35_last_error().decode())
    return int(n)


_ws_cache = {}  # (device index, stream) -> (bytes, address, tensor)


def _workspace(dev, nbytes, stream):
    """(address, owner) of one growing scratch buffer per (device, stream), owned by the Python host (the library itself never
    allocates); roles running concurrently on different streams must not share scratch"""
    got = _ws_cache.get((dev, stream))
    if got is None or got[0] < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=torch.device("cuda", dev))
        got = _ws_cache[dev, stream] = (buf.numel(), buf.data_ptr(), buf)
    return got[1], got[2]


def _scratch(dev, nbytes, stream):
    """(address, owner) of a call's workspace on `stream`.  While that stream captures a CUDA graph it comes from the graph's
    own memory: a graph must not hold the address of a buffer that a later, larger call replaces, nor share one with
    another graph that may be replayed beside it.  (torch's captures: a host that captures by other means brings its own
    workspace.)"""
    if stream != _raw_stream(dev) or dev != torch.cuda.current_device():
        # whether it captures, where the memory comes from and when it may go to somebody else are the stream's own matter
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, dev) if stream else torch.cuda.default_stream(dev)):
            return _scratch_here(dev, nbytes, stream)
    return _scratch_here(dev, nbytes, stream)


def _scratch_here(dev, nbytes, stream):
    if torch.cuda.is_current_stream_capturing():
        own = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", dev))
        return own.data_ptr(), own
    return _workspace(dev, nbytes, stream)


class _Plan:
    """What a call signature (role, names, dtypes, shapes) always binds: the IO table with everything but the pointers,
    and the scratch the role needs.  `workspace`, when the role needs it and the caller brings none, is the last entry."""

    def __init__(self, role, tensors):
        self.role = role.encode()
        self.need = workspace_bytes(role, **tensors) if "workspace" not in tensors else 0
        if self.need:
            tensors = dict(tensors, workspace=torch.empty(self.need, dtype=torch.uint8, device="meta"))
        arr, self.names = _table(tensors)  # the table points at these names
        self.n = len(tensors)
        self.bytes = bytes(arr)
        self.words = ctypes.c_uint64 * (len(self.bytes) // 8)


_IO_WORDS, _PTR_WORD = ctypes.sizeof(_IO) // 8, _IO.ptr.offset // 8
_plans = {}
# the handle of a device's current stream without the Stream object around it (1.2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def run_checked(role, stream=None, **tensors):
    """run() in Python: every check by name, for the calls that binding/bind.cc passes on and where it is not built.  The
    IO table of a signature is built once and copied per call."""
    L = lib()
    ts = tensors.values()
    devices = {t.get_device() for t in ts}
    if len(devices) != 1 or -1 in devices:
        if not devices or -1 in devices:
            raise ValueError("all tensors must live on the GPU (the library has no CPU path)")
        raise ValueError(f"the tensors are on different GPUs: {sorted(devices)}")
    dev, = devices
    sig = (role, tuple(tensors), tuple([t.dtype for t in ts]), tuple([t.shape for t in ts]))
    if False in [t.is_contiguous() for t in ts]:
        _table(tensors)  # names the tensor in its error
    plan = _plans.get(sig)
    if plan is None:
        if len(_plans) >= 4096:  # shapes of a long-running server: page tables grow by the page
            _plans.clear()
        plan = _plans[sig] = _Plan(role, tensors)
    ptrs = [t.data_ptr() for t in ts]
    if stream is None:
        stream = _raw_stream(dev)
    if plan.need:
        address, owner = _scratch(dev, plan.need, stream)  # owned until the call is issued: another thread may need more
        ptrs.append(address)
    table = plan.words.from_buffer_copy(plan.bytes)
    i = _PTR_WORD
    for p in ptrs:
        table[i] = p
        i += _IO_WORDS
    if dev == torch.cuda.current_device():
        _check(L.q35_run(plan.role, table, plan.n, stream))
    else:
        with torch.cuda.device(dev):
            _check(L.q35_run(plan.role, table, plan.n, stream))


_fast = None


def _fast_run():
    """binding/bind.cc's run, or run_checked where it was not built for this torch"""
    try:
        from . import _bind
    except ImportError:
        return run_checked
    if getattr(_bind, "built_for", None) != torch.__version__:  # it would read another torch's tensors
        return run_checked
    L = lib()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
    _bind.init(address(L.q35_run), address(L.q35_workspace_bytes), run_checked, _scratch, _check)
    return _bind.run


def run(role, stream=None, **tensors):
    """q35_run(role, ...) with the given tensors bound by name; a `workspace` is added when the role needs one.  The
    tensors are contiguous and on one GPU; the call goes to its current stream, or to the one given (a cudaStream_t as an
    integer).  The first call replaces this function in the module by its fast form."""
    global _fast, run
    if _fast is None:
        _fast = run = _fast_run()
    return _fast(role, stream, **tensors)


def io_table(role):
    L = lib()
    n = L.q35_io_table(role.encode(), None, 0)
    if n < 0:
        raise Q35Error(-n, L.q35_last_error().decode())
    buf = ctypes.create_string_buffer(n + 1)
    L.q35_io_table(role.encode(), buf, n + 1)
    return json.loads(buf.value.decode())


def roles():
    L = lib()
    return [L.q35_role_name(i).decode() for i in range(L.q35_role_count())]


def device_status(stream=None):
    if stream is None:
        stream = torch.cuda.current_stream().cuda_stream
    return lib().q35_device_status(ctypes.c_void_p(stream))
