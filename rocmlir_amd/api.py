"""ctypes binding of librocmlir_amd.so and torch-tensor front ends.

The option strings built here use the reference's own flag names
(rocmlir-gen.cpp:90-561 for gemm / attention, ConvGenerator.cpp:492-661 for
convolution), so a problem reads the same as on a rocmlir-gen command line.
"""
import contextlib
import ctypes as C
import os
import threading

_PKG = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_PKG, "librocmlir_amd.so")
_lib = None
_lock = threading.Lock()

MIIR_SUCCESS = 0
MIIR_INVALID_PARAM = 1
MIIR_INVALID_MODULE = 2
MIIR_BUILD_FAILURE = 3


class RockError(RuntimeError):
    pass


def library_path():
    return _LIB_PATH


def load_library():
    """Loads librocmlir_amd.so; raises RockError when it has not been built."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(_LIB_PATH):
            raise RockError(
                "librocmlir_amd.so is missing (%s): run "
                "`python -c 'import __graft_entry__ as g; g.build()'` "
                "or `python -m rocmlir_amd._build`" % _LIB_PATH)
        L = C.CDLL(_LIB_PATH)
        vp, sz = C.c_void_p, C.c_size_t
        L.miirCreateHandle.restype = vp
        L.miirCreateHandle.argtypes = [C.c_char_p]
        for name in ("miirGetKernelCount", "miirGetWorkspaceSize",
                     "miirLowerTuningParams", "miirLowerBin",
                     "miirDestroyHandle"):
            getattr(L, name).restype = C.c_int
            getattr(L, name).argtypes = [vp]
        L.rockamdGetWorkspaceSize64.restype = sz
        L.rockamdGetWorkspaceSize64.argtypes = [vp]
        L.rockamdGetArgumentInfo.restype = C.c_int
        L.rockamdGetArgumentInfo.argtypes = [vp, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int),
                                             C.POINTER(C.c_int64)]
        L.miirBufferGet.restype = C.c_int
        L.miirBufferGet.argtypes = [vp, C.c_char_p, C.POINTER(sz)]
        L.miirGetExecutionDims.restype = C.c_int
        L.miirGetExecutionDims.argtypes = [vp, C.POINTER(sz), C.POINTER(sz)]
        L.rockamdGetKernelName.restype = C.c_int
        L.rockamdGetKernelName.argtypes = [vp, C.c_char_p, C.POINTER(sz)]
        L.rockamdGetKernelAttrs.restype = C.c_int
        L.rockamdGetKernelAttrs.argtypes = [vp, C.POINTER(C.c_uint32)]
        L.rockamdGetKernelArgs.restype = C.c_int
        L.rockamdGetKernelArgs.argtypes = [vp, C.POINTER(C.c_int), vp,
                                           C.POINTER(sz)]
        L.rockamdGetPerfConfig.restype = sz
        L.rockamdGetPerfConfig.argtypes = [vp, C.c_char_p, sz]
        L.rockamdGetProblemKey.restype = sz
        L.rockamdGetProblemKey.argtypes = [vp, C.c_char_p, sz]
        L.rockamdSetScale.restype = C.c_int
        L.rockamdSetScale.argtypes = [vp, C.c_float]
        L.rockamdSetZeroPoint.restype = C.c_int
        L.rockamdSetZeroPoint.argtypes = [vp, C.c_int32]
        L.rockamdLaunch.restype = C.c_int
        L.rockamdLaunch.argtypes = [vp, C.POINTER(vp), C.c_int, vp]
        L.rockamdLaunchStaticWorkspace.restype = C.c_int
        L.rockamdLaunchStaticWorkspace.argtypes = [vp, C.POINTER(vp), C.c_int, vp]
        L.rockamdBenchmark.restype = C.c_int
        L.rockamdBenchmark.argtypes = [vp, C.POINTER(vp), C.c_int, vp, C.c_int,
                                       C.c_int, C.POINTER(C.c_float)]
        L.rockamdMeasureMfmaRate.restype = C.c_int
        L.rockamdMeasureMfmaRate.argtypes = [C.c_int, C.c_int, vp,
                                             C.POINTER(C.c_double)]
        L.rockamdGetLastError.restype = C.c_char_p
        L.rockamdGetLastError.argtypes = []
        L.rockamdTuningSpaceCreate.restype = vp
        L.rockamdTuningSpaceCreate.argtypes = [vp, C.c_int]
        L.rockamdTuningGetNumParams.restype = C.c_uint
        L.rockamdTuningGetNumParams.argtypes = [vp]
        L.rockamdTuningParamToString.restype = sz
        L.rockamdTuningParamToString.argtypes = [vp, C.c_uint, C.c_char_p, sz]
        L.rockamdTuningSpaceDestroy.restype = None
        L.rockamdTuningSpaceDestroy.argtypes = [vp]
        L.rockamdTuningSetFromStr.restype = C.c_int
        L.rockamdTuningSetFromStr.argtypes = [vp, C.c_char_p]
        L.rockamdTuningTableCreate.restype = vp
        L.rockamdTuningTableCreate.argtypes = []
        L.rockamdTuningTableDestroy.restype = None
        L.rockamdTuningTableDestroy.argtypes = [vp]
        L.rockamdTuningUpdateTable.restype = C.c_int
        L.rockamdTuningUpdateTable.argtypes = [vp, C.c_char_p, C.c_char_p,
                                               C.c_float]
        L.rockamdTuningSetFromTable.restype = C.c_int
        L.rockamdTuningSetFromTable.argtypes = [vp, vp]
        L.rockamdGetPointerMap.restype = C.c_int
        L.rockamdGetPointerMap.argtypes = [vp, C.POINTER(C.c_int),
                                           C.POINTER(C.c_int),
                                           C.POINTER(C.c_int32),
                                           C.POINTER(C.c_int64)]
        L.rockamdCheckArgumentSizes.restype = C.c_int
        L.rockamdCheckArgumentSizes.argtypes = [vp, C.POINTER(sz), C.c_int]
        L.rockamdGetParamPointers.restype = C.c_int
        L.rockamdGetParamPointers.argtypes = [vp, C.POINTER(C.c_int), C.POINTER(C.c_int32), C.POINTER(C.c_int32)]
        L.rockamdIsFusible.restype = C.c_int
        L.rockamdIsFusible.argtypes = [vp, C.c_char_p]
        L.rockamdGetNumPrefillArgs.restype = sz
        L.rockamdGetNumPrefillArgs.argtypes = [vp]
        L.rockamdGetPrefillArgsInfo.restype = None
        L.rockamdGetPrefillArgsInfo.argtypes = [vp, C.POINTER(sz), C.POINTER(C.c_float), sz]
        L.rockamdIsSplitKFaster.restype = C.c_int
        L.rockamdIsSplitKFaster.argtypes = [C.c_int64] * 5 + [C.c_int]
        _lib = L
        return _lib


def last_error():
    return load_library().rockamdGetLastError().decode()


_DTYPE_CODES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "fp8": 4}


def mfma_rate(dtype, random_data=False, stream=None):
    """Sustained 32x32 MFMA issue rate in TFLOP/s (TOP/s) on the current GPU
    for operand type `dtype`, with constant or hashed operand bits."""
    out = C.c_double(0)
    rc = load_library().rockamdMeasureMfmaRate(
        _DTYPE_CODES[dtype], int(bool(random_data)),
        getattr(stream, "cuda_stream", stream), C.byref(out))
    if rc != 0:
        raise RockError("rate probe failed (hip error %d): %s" % (rc, last_error()))
    return out.value


class RockKernel:
    """One problem -> one launchable kernel (a MiirHandle).

    Follows the reference client's call order (rocmlir-lib-test.cpp:31-96):
    create, lower tuning params, lower bin, read the binary and the launch
    dimensions."""

    def __init__(self, options):
        L = load_library()
        self.options = options
        self._h = L.miirCreateHandle(options.encode())
        if not self._h:
            raise RockError("miirCreateHandle failed: %s [%s]"
                            % (last_error(), options))
        self._refresh()

    def _refresh(self):
        """(Re)reads what describes the resolved kernel; called after
        creation and after a perf_config has been applied."""
        L = load_library()
        if L.miirLowerTuningParams(self._h) != MIIR_SUCCESS:
            raise RockError("miirLowerTuningParams failed")
        if L.miirLowerBin(self._h) != MIIR_SUCCESS:
            raise RockError("miirLowerBin failed")
        attrs = (C.c_uint32 * 2)()
        L.rockamdGetKernelAttrs(self._h, attrs)
        self.block_size, self.grid_size = int(attrs[0]), int(attrs[1])
        n = C.c_size_t(0)
        L.rockamdGetKernelName(self._h, None, C.byref(n))
        buf = C.create_string_buffer(n.value)
        L.rockamdGetKernelName(self._h, buf, C.byref(n))
        self.kernel_name = buf.value.decode()
        npt, psz = C.c_int(0), C.c_size_t(0)
        L.rockamdGetKernelArgs(self._h, C.byref(npt), None, C.byref(psz))
        self.num_pointers = npt.value
        self.params_size = psz.value
        # multi-kernel problems: kernels of the problem, its workspace, and the
        # caller pointer list every one of its kernels is launched with
        self.kernel_count = L.miirGetKernelCount(self._h)
        self.workspace_bytes = L.rockamdGetWorkspaceSize64(self._h)
        ncall = C.c_int(0)
        L.rockamdGetPointerMap(self._h, C.byref(ncall), None, None, None)
        self.caller_pointers = ncall.value
        self._pointers = C.c_void_p * ncall.value

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib is not None:
            _lib.miirDestroyHandle(h)

    # ---- description ------------------------------------------------------
    def _string(self, fn):
        buf = C.create_string_buffer(2048)
        n = fn(self._h, buf, 2048)
        if n == C.c_size_t(-1).value:
            raise RockError("string query failed")
        return buf.value.decode()

    @property
    def perf_config(self):
        return self._string(load_library().rockamdGetPerfConfig)

    @property
    def problem_key(self):
        return self._string(load_library().rockamdGetProblemKey)

    def code_object(self):
        L = load_library()
        n = C.c_size_t(0)
        if L.miirBufferGet(self._h, None, C.byref(n)) != MIIR_SUCCESS:
            raise RockError("miirBufferGet(size) failed")
        buf = C.create_string_buffer(n.value)
        if L.miirBufferGet(self._h, buf, C.byref(n)) != MIIR_SUCCESS:
            raise RockError("miirBufferGet failed")
        return buf.raw[:n.value]

    def params(self):
        L = load_library()
        n = C.c_size_t(self.params_size)
        buf = C.create_string_buffer(n.value)
        npt = C.c_int(0)
        L.rockamdGetKernelArgs(self._h, C.byref(npt), buf, C.byref(n))
        return buf.raw

    def execution_dims(self):
        g, l = C.c_size_t(0), C.c_size_t(0)
        rc = load_library().miirGetExecutionDims(self._h, C.byref(g),
                                                 C.byref(l))
        if rc != MIIR_SUCCESS:
            raise RockError("miirGetExecutionDims failed (%d)" % rc)
        return g.value, l.value

    # ---- tuning (mlir-c/Dialect/Rock.h:39-117) -------------------------------
    TUNING_KINDS = {"quick": 0, "full": 1, "exhaustive": 2}

    def tuning_space(self, kind="full"):
        """perf_config strings of the kernels this problem can run on; the
        first is the built-in table's choice.  kind: "quick" (at most three
        entries), "full" (every kernel) or "exhaustive" (RockEnums.h:19-23)."""
        L = load_library()
        sp = L.rockamdTuningSpaceCreate(self._h, self.TUNING_KINDS[kind])
        if not sp:
            raise RockError("rockamdTuningSpaceCreate failed")
        try:
            out = []
            for i in range(L.rockamdTuningGetNumParams(sp)):
                buf = C.create_string_buffer(128)
                n = L.rockamdTuningParamToString(sp, i, buf, 128)
                if n == C.c_size_t(-1).value or n >= 128:
                    raise RockError("rockamdTuningParamToString failed")
                out.append(buf.value.decode())
            return out
        finally:
            L.rockamdTuningSpaceDestroy(sp)

    def set_perf_config(self, perf_config):
        """Re-resolves the kernel under `perf_config`
        (mlirRockTuningSetFromStr); unknown strings fall back to the table."""
        if not load_library().rockamdTuningSetFromStr(self._h,
                                                      perf_config.encode()):
            raise RockError("rockamdTuningSetFromStr(%r) failed: %s"
                            % (perf_config, last_error()))
        self._refresh()

    def arguments(self):
        """[(dtype code, dims)] for every pointer launch() takes (rockamdGetArgumentInfo)."""
        out = []
        for i in range(self.caller_pointers):
            dt, rank, dims = C.c_int(), C.c_int(), (C.c_int64 * 6)()
            if load_library().rockamdGetArgumentInfo(self._h, i, C.byref(dt), C.byref(rank), dims) != 0:
                raise RockError("rockamdGetArgumentInfo(%d) failed" % i)
            out.append((dt.value, list(dims[:rank.value])))
        return out

    def set_scale(self, scale):
        load_library().rockamdSetScale(self._h, float(scale))

    def set_zero_point(self, zp):
        load_library().rockamdSetZeroPoint(self._h, int(zp))

    # ---- launch --------------------------------------------------------------
    def _check_sizes(self, args):
        """Every tensor argument must hold at least the bytes the kernel list addresses in it
        (rockamdCheckArgumentSizes): a short one is an error here, not a fault on the device."""
        sizes = (C.c_size_t * len(args))()
        for i, a in enumerate(args):
            sizes[i] = 0 if a is None or isinstance(a, int) else a.numel() * a.element_size()
        if load_library().rockamdCheckArgumentSizes(self._h, sizes, len(args)) != MIIR_SUCCESS:
            raise RockError("%s: %s" % (self.kernel_name, last_error()))

    def _pointer_array(self, args):
        if len(args) != self.caller_pointers:
            raise RockError("kernel %s takes %d pointer arguments, got %d"
                            % (self.kernel_name, self.caller_pointers, len(args)))
        self._check_sizes(args)
        arr = (C.c_void_p * len(args))()
        for i, a in enumerate(args):
            if a is None:
                arr[i] = None
            elif isinstance(a, int):
                arr[i] = a
            else:  # torch tensor
                if not a.is_cuda:
                    raise RockError("tensor arguments must live on the GPU")
                arr[i] = a.data_ptr()
        return arr

    @staticmethod
    def _stream(stream):
        if stream is None:
            import torch
            return torch.cuda.current_stream().cuda_stream
        return getattr(stream, "cuda_stream", stream)

    def launch(self, *args, stream=None):
        arr = self._pointer_array(args)
        rc = load_library().rockamdLaunch(self._h, arr, len(args),
                                          self._stream(stream))
        if rc != 0:
            raise RockError("launch of %s failed (hip error %d): %s"
                            % (self.kernel_name, rc, last_error()))

    def launch_checked(self, args):
        """launch() on torch's current stream for a caller that has checked the tensors against the problem's sizes,
        that they are on one device and that this device is the current one: a call costs the host a third of
        launch()."""
        if torch is None:
            _load_torch()
        if not args[0].is_cuda:
            raise RockError("tensor arguments must live on the GPU")
        arr = self._pointers(*[None if a is None else a.data_ptr() for a in args])
        rc = _lib.rockamdLaunch(self._h, arr, self.caller_pointers,
                                torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))
        if rc != 0:
            raise RockError("launch of %s failed (hip error %d): %s" % (self.kernel_name, rc, last_error()))

    def benchmark(self, *args, warmup=3, iters=20, stream=None):
        """Average milliseconds per launch (HIP events on the launch stream)."""
        arr = self._pointer_array(args)
        ms = C.c_float(0)
        rc = load_library().rockamdBenchmark(self._h, arr, len(args),
                                             self._stream(stream), warmup,
                                             iters, C.byref(ms))
        if rc != 0:
            raise RockError("benchmark of %s failed (hip error %d): %s"
                            % (self.kernel_name, rc, last_error()))
        return ms.value


class RockProgram:
    """All kernels of one problem (miirGetKernelCount handles, one per
    --kernel_id) plus the workspace they share; launch() runs them in order
    on one stream.  Single-kernel problems behave like their RockKernel."""

    def __init__(self, options):
        self.options = options
        self.lock = threading.Lock()   # a handle must not be used from two threads at once
        self._build(options)

    def _build(self, options):
        first = RockKernel(options)
        self.kernels = [first] + [RockKernel("%s --kernel_id %d" % (options, i))
                                  for i in range(1, first.kernel_count)]
        self.workspace_bytes = first.workspace_bytes
        self._workspace = None

    @property
    def main(self):
        """The contraction kernel: the last GEMM, convolution or attention kernel of the list (conversion
        kernels may run in front of it, the reduction of split partial sums behind it)."""
        for k in reversed(self.kernels):
            if k.kernel_name.startswith(("rock_gemm_", "rock_conv_", "rock_attention_", "rock_token_gemm_")):
                return k
        return self.kernels[-1]

    # what rocmlir_amd.tuning.tune() uses, so that problems of several kernels tune like single ones
    kernel_name = property(lambda self: self.main.kernel_name)
    perf_config = property(lambda self: self.main.perf_config)
    problem_key = property(lambda self: self.main.problem_key)

    def tuning_space(self, kind="full"):
        return self.kernels[0].tuning_space(kind)

    def set_perf_config(self, perf_config):
        """Plans the problem again under `perf_config` (the kernel list can
        change: a request may add or drop conversion kernels)."""
        self._build(self.options + (" --perf_config %s" % perf_config if perf_config else ""))

    def _args(self, args):
        if self.kernels[0].caller_pointers == len(args):
            return args   # no workspace pointer in this problem's caller list
        if self._workspace is None:
            import torch
            dev = next(a.device for a in args if a is not None and not isinstance(a, int))
            self._workspace = torch.empty(max(self.workspace_bytes, 16), dtype=torch.uint8, device=dev)
        return tuple(args) + (self._workspace,)

    def launch(self, *args, stream=None):
        full = self._args(args)
        for k in self.kernels:
            k.launch(*full, stream=stream)

    def benchmark(self, *args, warmup=3, iters=20, stream=None):
        """Sum of the kernels' average times in milliseconds."""
        return sum(ms for _, ms in self.benchmark_each(*args, warmup=warmup, iters=iters, stream=stream))

    def benchmark_sequence(self, *args, warmup=2, iters=5):
        """Average milliseconds for the whole list launched in order, back to back (events on torch's current
        stream, where launch() puts the kernels): what a caller of a many-kernel problem waits for, gaps between
        the kernels and the state of the caches they leave each other included."""
        import torch
        full = self._args(args)
        for _ in range(warmup):
            self.launch(*args)
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(iters):
            for k in self.kernels:
                k.launch(*full)
        stop.record()
        stop.synchronize()
        return start.elapsed_time(stop) / iters

    def benchmark_each(self, *args, warmup=3, iters=20, stream=None):
        """[(kernel name, average time in milliseconds)] in launch order."""
        full = self._args(args)
        return [(k.kernel_name, k.benchmark(*full, warmup=warmup, iters=iters, stream=stream)) for k in self.kernels]


# ---------------------------------------------------------------------------
# torch front ends
# ---------------------------------------------------------------------------
_kernel_cache = {}


def _kernel(options):
    k = _kernel_cache.get(options)
    if k is None:
        k = _kernel_cache[options] = RockKernel(options)
    return k


_program_cache = {}


def _program(options):
    p = _program_cache.get(options)
    if p is None:
        p = _program_cache[options] = RockProgram(options)
    return p


_dtype_names, _torch_dtypes = {}, {}


def _dtype_tables():
    import torch
    names = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "i32": torch.int32}
    if hasattr(torch, "float8_e4m3fn"):
        names["fp8"], names["bf8"] = torch.float8_e4m3fn, torch.float8_e5m2
    _torch_dtypes.update(names)
    _dtype_names.update({v: k for k, v in names.items()})


def _dtype_name(dt):
    if not _dtype_names:
        _dtype_tables()
    try:
        return _dtype_names[dt]
    except KeyError:
        raise RockError("unsupported tensor dtype %s" % dt)


def _torch_dtype(name):
    if not _torch_dtypes:
        _dtype_tables()
    return _torch_dtypes[name]


def _is_tensor(x):
    return hasattr(x, "data_ptr")


def _channel_vectors(scale, zero_point, quant_scale, out_zero_point):
    """The per-channel quantisation vectors among the four epilogue values, in
    the order the library takes them behind the problem's own tensors, and the
    flags that announce them (a torch tensor instead of a number means one
    value per output channel: f32 scales, int32 or int8 zero points)."""
    import torch
    flags, vectors = "", []
    for name, val, is_zp in (("scale_vector", scale, False), ("zero_point_vector", zero_point, True),
                             ("quant_scale_vector", quant_scale, False),
                             ("out_zero_point_vector", out_zero_point, True)):
        if not _is_tensor(val):
            continue
        if is_zp:
            if val.dtype not in (torch.int8, torch.int32):
                raise RockError("%s: int32 or int8 elements" % name)
            flags += " -%s %s" % (name, "i8" if val.dtype == torch.int8 else "i32")
        else:
            if val.dtype != torch.float32:
                raise RockError("%s: f32 elements" % name)
            flags += " -%s true" % name
        vectors.append(val.contiguous())
    return flags, vectors


def _epilogue_flags(scale, zero_point, bias, relu, quant_scale, out_zero_point,
                    activation=None, clip=None, residual=None, residual_op="add"):
    s = ""
    if scale is not None and not _is_tensor(scale):
        s += " -scale %.9g" % scale
    if not _is_tensor(zero_point) and zero_point:
        s += " -zero_point %d" % zero_point
    if quant_scale is not None and not _is_tensor(quant_scale):
        s += " -quant_scale %.9g" % quant_scale
    if not _is_tensor(out_zero_point) and out_zero_point:
        s += " -out_zero_point %d" % out_zero_point
    s += _channel_vectors(scale, zero_point, quant_scale, out_zero_point)[0]
    if bias is not None:
        s += " -bias true"
    if relu:
        s += " -relu true"
    if activation:
        s += " -activation %s" % activation
    if clip is not None:
        s += " -activation clip -clip_min %.9g -clip_max %.9g" % tuple(clip)
    if residual is not None:
        s += " -residual %s" % residual_op
    return s


def gemm(a, b, *, transA=False, transB=False, transC=False, out_dtype=None,
         scale=None, zero_point=0, bias=None, relu=False, quant_scale=None,
         out_zero_point=0, activation=None, clip=None, residual=None,
         residual_op="add", out=None, perf_config=None, stream=None,
         info=None, split_k=True, layout_conversion=True, accumulate=False,
         token_scale=None):
    """C = epilogue(A x B) with the reference's storage conventions
    (rocmlir-gen.cpp:2058-2080): a is [G,M,K] ([G,K,M] if transA), b is
    [G,K,N] ([G,N,K] if transB), result [G,M,N] ([G,N,M] if transC).
    2-D inputs mean G = 1.  `scale`, `zero_point`, `quant_scale` and
    `out_zero_point` are numbers (per tensor) or torch tensors with one element
    per column of the result (per channel: f32 scales, int32 / int8 zero
    points).  The epilogue runs scale / zero point, per-column
    `bias`, `residual` (a tensor shaped and typed like the result, combined by
    `residual_op` "add" or "mul"), then `activation` ("relu", "sigmoid",
    "tanh", "erf", "gelu", "exp") or `clip=(lo, hi)`, then the narrowing to
    the output type.  A dict passed as `info` receives the name and
    perf_config of the GEMM kernel that ran and the names of all kernels of
    the problem (operands that are not whole 16-byte chunks are first copied
    into padded ones unless `layout_conversion` is False; a long reduction
    over few output tiles is split over blocks unless `split_k` is False).
    `accumulate=True` (rocmlir-gen's -store-method atomic_add) adds the
    result into `out` instead of overwriting it.

    `token_scale` (int8 operands, G = 1): a float32 tensor with one value per
    row of the result, as quantize_tokens() returns it; the result is
    (sum - zero_point) * scale[n] * token_scale[m] (+ bias, then relu or clip)
    in `out_dtype` f16 (the default), bf16 or f32.  K up to 131071; no transA,
    transC, residual, requantisation or accumulation beside it."""
    if token_scale is not None:
        if transA or transC or accumulate or residual is not None or quant_scale is not None or _is_tensor(zero_point) \
                or _is_tensor(out_zero_point) or out_zero_point:
            raise RockError("gemm: token_scale takes scale, a scalar zero_point, bias, relu and clip only")
        return _token_scaled_gemm(a, b, transB, out_dtype, scale, zero_point, bias, relu, activation, clip, out,
                                  perf_config, stream, info, token_scale)
    import torch
    if accumulate and (out is None or residual is not None):
        raise RockError("gemm: accumulate=True adds into `out` and takes no residual")
    a3 = a if a.dim() == 3 else a.unsqueeze(0)
    b3 = b if b.dim() == 3 else b.unsqueeze(0)
    a3, b3 = a3.contiguous(), b3.contiguous()
    G = a3.shape[0]
    M, K = (a3.shape[2], a3.shape[1]) if transA else (a3.shape[1], a3.shape[2])
    Kb, N = (b3.shape[2], b3.shape[1]) if transB else (b3.shape[1], b3.shape[2])
    if Kb != K or b3.shape[0] != G:
        raise RockError("gemm: operand shapes do not match")
    ta, tb = _dtype_name(a3.dtype), _dtype_name(b3.dtype)
    t = ta if ta == tb else "%s_%s" % (ta, tb)
    opts = ("-operation gemm -arch gfx950 -t %s -g %d -m %d -n %d -k %d"
            " -transA %s -transB %s -transC %s"
            % (t, G, M, N, K, str(bool(transA)).lower(),
               str(bool(transB)).lower(), str(bool(transC)).lower()))
    if out_dtype is not None:
        opts += " -out_datatype %s" % out_dtype
    if perf_config:
        opts += " -perf_config %s" % perf_config
    if not split_k:
        opts += " -split_k false"
    if not layout_conversion:
        opts += " -layout_conversion false"
    if accumulate:
        opts += " -store-method atomic_add"
    opts += _epilogue_flags(scale, zero_point, bias, relu, quant_scale,
                            out_zero_point, activation, clip, residual,
                            residual_op)
    prog = _program(opts)   # one kernel, or several: padded operand copies, a reduction split over blocks
    k = next(x for x in prog.kernels if x.kernel_name.startswith("rock_gemm_"))
    if info is not None:
        info["kernel_name"] = k.kernel_name
        info["perf_config"] = k.perf_config
        info["kernels"] = [x.kernel_name for x in prog.kernels]
    if out_dtype is None:
        out_dtype = {"i8": "i32", "fp8": "f32", "bf8": "f32"}.get(ta, ta)
    shape = (G, N, M) if transC else (G, M, N)
    if out is None:
        out = torch.empty(shape, dtype=_torch_dtype(out_dtype), device=a.device)
    vectors = _channel_vectors(scale, zero_point, quant_scale, out_zero_point)[1]
    if any(v.numel() != N for v in vectors):
        raise RockError("gemm: a per-channel vector holds one element per column of the result")
    if residual is None:
        prog.launch(a3, b3, out, bias, *vectors, stream=stream)
    else:
        if residual.dtype != out.dtype or residual.numel() != out.numel():
            raise RockError("gemm: the residual must have the result's type and size")
        prog.launch(a3, b3, out, bias, residual.contiguous(), *vectors, stream=stream)
    return out if a.dim() == 3 else out.squeeze(0)


def conv2d(fil, inp, *, fil_layout, in_layout, out_layout, batchsize,
           in_channels, out_channels, in_h, in_w, fil_h, fil_w, groupsize=1,
           stride=(1, 1), padding=(0, 0), dilation=(1, 1), out_dtype=None,
           scale=None, zero_point=0, bias=None, relu=False, quant_scale=None,
           out_zero_point=0, activation=None, clip=None, residual=None,
           residual_op="add", out=None, perf_config=None, stream=None,
           info=None, padding_r=None, layout_conversion=True):
    """Forward convolution; tensors are flat device buffers laid out as the
    layout strings say (Miir / rocmlir-gen spelling, e.g. 'gkyxc', 'nhwgc',
    'NGCHW').  Epilogue arguments as for gemm(); the residual is laid out
    like the output.  `padding` is the top / left padding and, unless
    `padding_r` gives the bottom / right one (--padding_h_r / --padding_w_r),
    that one too.  Returns the flat output tensor.  A dict passed as `info`
    receives the name and perf_config of the kernel that ran.
    `layout_conversion=False` keeps the tensors where they lie (no conversion
    kernels in front; the element-wise kernel where the vector ones cannot read them)."""
    import torch
    t = _dtype_name(inp.dtype)
    pr = padding if padding_r is None else padding_r
    ho = (in_h + padding[0] + pr[0] - (fil_h - 1) * dilation[0] - 1) // stride[0] + 1
    wo = (in_w + padding[1] + pr[1] - (fil_w - 1) * dilation[1] - 1) // stride[1] + 1
    opts = ("--operation conv --arch gfx950 --in_type %s --fil_type %s"
            " --fil_layout %s --in_layout %s --out_layout %s --batchsize %d"
            " --groupsize %d --in_channels %d --out_channels %d --in_h %d"
            " --in_w %d --out_h %d --out_w %d --fil_h %d --fil_w %d"
            " --dilation_h %d --dilation_w %d --conv_stride_h %d"
            " --conv_stride_w %d --padding_h %d --padding_w %d"
            % (t, _dtype_name(fil.dtype), fil_layout, in_layout, out_layout,
               batchsize, groupsize, in_channels, out_channels, in_h, in_w, ho,
               wo, fil_h, fil_w, dilation[0], dilation[1], stride[0], stride[1],
               padding[0], padding[1]))
    if padding_r is not None:
        opts += " --padding_h_r %d --padding_w_r %d" % (pr[0], pr[1])
    if out_dtype is not None:
        opts += " --out_type %s" % out_dtype
    if perf_config:
        opts += " --perf_config %s" % perf_config
    if not layout_conversion:
        opts += " --layout_conversion false"
    opts += _epilogue_flags(scale, zero_point, bias, relu, quant_scale,
                            out_zero_point, activation, clip, residual,
                            residual_op)
    prog = _program(opts)
    k = prog.main
    if info is not None:
        info["kernel_name"] = k.kernel_name
        info["perf_config"] = k.perf_config
        info["kernels"] = [x.kernel_name for x in prog.kernels]
    if out_dtype is None:
        out_dtype = {"i8": "i32", "fp8": "f32", "bf8": "f32"}.get(t, t)
    if out is None:
        out = torch.empty(batchsize * out_channels * ho * wo,
                          dtype=_torch_dtype(out_dtype), device=inp.device)
    vectors = _channel_vectors(scale, zero_point, quant_scale, out_zero_point)[1]
    if any(v.numel() != out_channels for v in vectors):
        raise RockError("conv2d: a per-channel vector holds one element per output channel")
    if residual is None:
        prog.launch(fil.contiguous(), inp.contiguous(), out, bias, *vectors, stream=stream)
    else:
        if residual.dtype != out.dtype or residual.numel() != out.numel():
            raise RockError("conv2d: the residual must have the output's type and size")
        prog.launch(fil.contiguous(), inp.contiguous(), out, bias, residual.contiguous(), *vectors, stream=stream)
    return out


def attention(q, k, v, *, scale=1.0, bias=None, scale_tensor=None, mask=None, other=None, zero_point=0,
              transQ=False, transK=False, transV=False, transO=False, out=None, stream=None, info=None,
              score_workspace_limit=None, program=None, inputs=(), layout_conversion=True):
    """O = softmax(scale * scale_tensor * Q K + bias) V (bias and scale_tensor
    optional [G,seq_q,seq_k] tensors, rocmlir-gen's -with-attn-bias /
    -with-attn-scale).  `mask` (int8 or bool, [G,seq_q,seq_k]) with `other`
    (same shape, v's type) puts migraphx.where(mask, scores, other) in front of
    the softmax (mixr-attn-where.mlir:11): a zero in the mask replaces the score
    by other's element.  Storage follows the reference's
    conventions (rocmlir-gen.cpp:2149-2200): q [G,seq_q,d] ([G,d,seq_q] if
    transQ); k [G,d,seq_k] ([G,seq_k,d] if transK -- the usual row-major keys);
    v [G,seq_k,dv] ([G,dv,seq_k] if transV); result [G,seq_q,dv]
    ([G,dv,seq_q] if transO).  int8 q and k (with f16 v, bias, scale_tensor)
    select the quantised first GEMM: the scores are (acc - zero_point) * scale.
    A dict passed as `info` receives the names of the kernels that ran.
    `score_workspace_limit` (bytes) bounds the score chunk of the three-kernel
    form (f32, head dimensions above 256); the default is 32 MiB.
    `program` is a pre-softmax element-wise tree in postfix form over the score
    `x`, the tensors `inputs` (`t0`, `t1`, ...; each [G,seq_q,seq_k], any of
    f32 / f16 / bf16 / int8) and constants `c:<number>`, e.g.
    "x,t0,mul,exp,t1,add" (the region of rock.attention, RockOps.td:208-254);
    it replaces scale, bias, scale_tensor and mask."""
    import torch
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    G = q.shape[0]
    sq, dqk = (q.shape[2], q.shape[1]) if transQ else (q.shape[1], q.shape[2])
    sk = k.shape[1] if transK else k.shape[2]
    dv = v.shape[1] if transV else v.shape[2]
    t = _dtype_name(q.dtype)
    tf = lambda b: str(bool(b)).lower()  # noqa: E731
    opts = ("-operation attention -arch gfx950 -t %s -g %d -seq_len_q %d"
            " -seq_len_k %d -head_dim_qk %d -head_dim_v %d -transQ %s"
            " -transK %s -transV %s -transO %s -scale %.9g"
            % (t, G, sq, sk, dqk, dv, tf(transQ), tf(transK), tf(transV),
               tf(transO), scale))
    if bias is not None:
        opts += " -with-attn-bias true"
    if scale_tensor is not None:
        opts += " -with-attn-scale true"
    if zero_point:
        opts += " -zero_point %d" % zero_point
    if (mask is None) != (other is None):
        raise RockError("attention: mask and other come together")
    if mask is not None:
        opts += " -with-attn-mask true"
        if tuple(mask.shape) != (G, sq, sk) or tuple(other.shape) != (G, sq, sk) or other.dtype != v.dtype:
            raise RockError("attention: mask and other are [G, seq_q, seq_k]; other has v's type")
        mask = mask.to(torch.int8).contiguous()
    if not layout_conversion:   # no copies in front of or behind the kernel: tensors are read as they lie
        opts += " -layout_conversion false"
    if score_workspace_limit is not None:
        opts += " -score_workspace_limit %d" % score_workspace_limit
    if program:
        if bias is not None or scale_tensor is not None or mask is not None or scale != 1.0:
            raise RockError("attention: a program replaces scale, bias, scale_tensor and mask")
        opts += " -attn_elementwise %s" % program.replace(" ", "")
        if inputs:
            opts += " -attn_inputs %s" % ",".join(_dtype_name(t.dtype) for t in inputs)
    kern = _program(opts)   # one fused kernel, or three for head dimensions above 128 and f32
    if info is not None:
        info["kernels"] = [k.kernel_name for k in kern.kernels]
    shape = (G, dv, sq) if transO else (G, sq, dv)
    if out is None:
        out = torch.empty(shape, dtype=v.dtype, device=q.device)
    pre = ([] if scale_tensor is None else [scale_tensor.contiguous()]) + [bias]
    if mask is not None:
        pre += [mask, other.contiguous()]
    if program:
        pre = [t.contiguous() for t in inputs]
    kern.launch(q, k, v, *pre, out, stream=stream)
    return out


def conv3d(fil, inp, *, fil_layout, in_layout, out_layout, batchsize, in_channels, out_channels, in_size,
           fil_size, groupsize=1, stride=(1, 1, 1), padding=(0, 0, 0), dilation=(1, 1, 1), out_dtype=None,
           scale=None, zero_point=0, bias=None, relu=False, quant_scale=None, out_zero_point=0,
           activation=None, clip=None, residual=None, residual_op="add", out=None, perf_config=None,
           stream=None, info=None):
    """Forward convolution over three spatial dimensions.  Sizes, strides,
    padding and dilation are (h, w, d) triples; the layout strings have six
    letters ('ngc012' / 'gkc012' / 'ngk012' in rocmlir-gen's spelling, h w d
    and y x z accepted for 0 1 2).  Epilogue arguments as for conv2d(); the
    residual is laid out like the output.  Returns the flat output tensor."""
    import torch
    t = _dtype_name(inp.dtype)
    outs = [(in_size[a] + 2 * padding[a] - (fil_size[a] - 1) * dilation[a] - 1) // stride[a] + 1 for a in range(3)]
    opts = ("--operation conv --arch gfx950 --in_type %s --fil_type %s --fil_layout %s --in_layout %s"
            " --out_layout %s --batchsize %d --groupsize %d --in_channels %d --out_channels %d"
            % (t, _dtype_name(fil.dtype), fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
               out_channels))
    for a, s in enumerate("hwd"):
        opts += (" --in_%s %d --fil_%s %d --out_%s %d --dilation_%s %d --conv_stride_%s %d --padding_%s %d"
                 % (s, in_size[a], s, fil_size[a], s, outs[a], s, dilation[a], s, stride[a], s, padding[a]))
    if out_dtype is not None:
        opts += " --out_type %s" % out_dtype
    if perf_config:
        opts += " --perf_config %s" % perf_config
    opts += _epilogue_flags(scale, zero_point, bias, relu, quant_scale, out_zero_point, activation, clip, residual,
                            residual_op)
    prog = _program(opts)
    if info is not None:
        info["kernels"] = [x.kernel_name for x in prog.kernels]
        info["workspace_bytes"] = prog.workspace_bytes
    if out_dtype is None:
        out_dtype = {"i8": "i32", "fp8": "f32", "bf8": "f32"}.get(t, t)
    if out is None:
        out = torch.empty(batchsize * out_channels * outs[0] * outs[1] * outs[2], dtype=_torch_dtype(out_dtype),
                          device=inp.device)
    if residual is None:
        prog.launch(fil.contiguous(), inp.contiguous(), out, bias, stream=stream)
    else:
        if residual.dtype != out.dtype or residual.numel() != out.numel():
            raise RockError("conv3d: the residual must have the output's type and size")
        prog.launch(fil.contiguous(), inp.contiguous(), out, bias, residual.contiguous(), stream=stream)
    return out


def _conv3d_options(operation, t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
                    out_channels, in_size, fil_size, stride, padding, dilation):
    opts = ("--operation %s --arch gfx950 --in_type %s --fil_type %s --out_type %s --fil_layout %s --in_layout %s"
            " --out_layout %s --batchsize %d --groupsize %d --in_channels %d --out_channels %d"
            % (operation, t, t, t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
               out_channels))
    for a, s in enumerate("hwd"):
        opts += (" --in_%s %d --fil_%s %d --dilation_%s %d --conv_stride_%s %d --padding_%s %d"
                 % (s, in_size[a], s, fil_size[a], s, dilation[a], s, stride[a], s, padding[a]))
    return opts


def conv3d_bwd_data(fil, dout, *, fil_layout, in_layout, out_layout, batchsize, in_channels, out_channels, in_size,
                    fil_size, groupsize=1, stride=(1, 1, 1), padding=(0, 0, 0), dilation=(1, 1, 1), out=None,
                    stream=None, info=None):
    """Gradient of conv3d with respect to its input (operation conv_bwd_data
    with the in_d / fil_d keys): `dout` is the gradient of the output, laid
    out as `out_layout` says; returns the flat input-shaped gradient."""
    import torch
    t = _dtype_name(dout.dtype)
    prog = _program(_conv3d_options("conv_bwd_data", t, fil_layout, in_layout, out_layout, batchsize, groupsize,
                                    in_channels, out_channels, in_size, fil_size, stride, padding, dilation))
    if info is not None:
        info["kernels"] = [k.kernel_name for k in prog.kernels]
        info["workspace_bytes"] = prog.workspace_bytes
    if out is None:
        out = torch.empty(batchsize * in_channels * in_size[0] * in_size[1] * in_size[2], dtype=dout.dtype,
                          device=dout.device)
    prog.launch(fil.contiguous(), out, dout.contiguous(), None, stream=stream)
    return out


def conv3d_bwd_weight(inp, dout, *, fil_layout, in_layout, out_layout, batchsize, in_channels, out_channels,
                      in_size, fil_size, groupsize=1, stride=(1, 1, 1), padding=(0, 0, 0), dilation=(1, 1, 1),
                      out=None, stream=None, info=None):
    """Gradient of conv3d with respect to its filter (operation
    conv_bwd_weight with the in_d / fil_d keys); returns the flat
    filter-shaped gradient."""
    import torch
    t = _dtype_name(dout.dtype)
    prog = _program(_conv3d_options("conv_bwd_weight", t, fil_layout, in_layout, out_layout, batchsize, groupsize,
                                    in_channels, out_channels, in_size, fil_size, stride, padding, dilation))
    if info is not None:
        info["kernels"] = [k.kernel_name for k in prog.kernels]
        info["workspace_bytes"] = prog.workspace_bytes
    if out is None:
        out = torch.empty(out_channels * (in_channels // groupsize) * fil_size[0] * fil_size[1] * fil_size[2],
                          dtype=dout.dtype, device=dout.device)
    prog.launch(out, inp.contiguous(), dout.contiguous(), None, stream=stream)
    return out


def _conv_options(operation, t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels, out_channels,
                  in_h, in_w, fil_h, fil_w, stride, padding, dilation):
    return ("--operation %s --arch gfx950 --in_type %s --fil_type %s --out_type %s"
            " --fil_layout %s --in_layout %s --out_layout %s --batchsize %d"
            " --groupsize %d --in_channels %d --out_channels %d --in_h %d"
            " --in_w %d --fil_h %d --fil_w %d --dilation_h %d --dilation_w %d"
            " --conv_stride_h %d --conv_stride_w %d --padding_h %d --padding_w %d"
            % (operation, t, t, t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
               out_channels, in_h, in_w, fil_h, fil_w, dilation[0], dilation[1], stride[0], stride[1],
               padding[0], padding[1]))


def conv2d_bwd_data(fil, dout, *, fil_layout, in_layout, out_layout, batchsize, in_channels, out_channels, in_h,
                    in_w, fil_h, fil_w, groupsize=1, stride=(1, 1), padding=(0, 0), dilation=(1, 1), out=None,
                    layout_conversion=True, stream=None, info=None):
    """Gradient of conv2d with respect to its input (rocmlir-gen / Miir
    operation conv_bwd_data): `dout` is the gradient of the output, laid out
    as `out_layout` says; returns the flat input-shaped gradient."""
    import torch
    t = _dtype_name(dout.dtype)
    opts = _conv_options("conv_bwd_data", t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
                         out_channels, in_h, in_w, fil_h, fil_w, stride, padding, dilation)
    if not layout_conversion:
        opts += " --layout_conversion false"
    prog = _program(opts)
    if info is not None:
        info["kernels"] = [k.kernel_name for k in prog.kernels]
        info["workspace_bytes"] = prog.workspace_bytes
    if out is None:
        out = torch.empty(batchsize * in_channels * in_h * in_w, dtype=dout.dtype, device=dout.device)
    prog.launch(fil.contiguous(), out, dout.contiguous(), None, stream=stream)
    return out


def conv2d_bwd_weight(inp, dout, *, fil_layout, in_layout, out_layout, batchsize, in_channels, out_channels, in_h,
                      in_w, fil_h, fil_w, groupsize=1, stride=(1, 1), padding=(0, 0), dilation=(1, 1), out=None,
                      layout_conversion=True, stream=None, info=None, as_gemm=True):
    """Gradient of conv2d with respect to its filter (operation
    conv_bwd_weight); returns the flat filter-shaped gradient.  as_gemm=False
    keeps channels-last problems off the single K-major GEMM over the tensors
    as they lie (--bwd_weight_gemm false)."""
    import torch
    t = _dtype_name(dout.dtype)
    opts = _conv_options("conv_bwd_weight", t, fil_layout, in_layout, out_layout, batchsize, groupsize, in_channels,
                         out_channels, in_h, in_w, fil_h, fil_w, stride, padding, dilation)
    if not layout_conversion:
        opts += " --layout_conversion false"
    if not as_gemm:
        opts += " --bwd_weight_gemm false"
    prog = _program(opts)
    if info is not None:
        info["kernels"] = [k.kernel_name for k in prog.kernels]
        info["workspace_bytes"] = prog.workspace_bytes
    if out is None:
        out = torch.empty(out_channels * (in_channels // groupsize) * fil_h * fil_w, dtype=dout.dtype,
                          device=dout.device)
    prog.launch(out, inp.contiguous(), dout.contiguous(), None, stream=stream)
    return out


# ---------------------------------------------------------------------------
# operators over the token rows of a language model (csrc/plan_tokens.cpp)
# ---------------------------------------------------------------------------
_token_plans = {}
torch = None   # the module, once one of these operators has been called


def _load_torch():
    global torch
    import torch as module
    torch = module


def _token_plan(names, *values):
    """The plan of a problem given as the names of its options (one string) and their values; None and False leave an
    option out.  The first two are the operation and the operands' type."""
    key = (names, values)
    p = _token_plans.get(key)
    if p is None:
        text = "-arch gfx950"
        for k, v in zip(names.split(), values):
            if v is not None and v is not False:
                text += " -%s %s" % (k, "true" if v is True else "%.9g" % v if isinstance(v, float) else v)
        p = RockProgram(text)
        if len(_token_plans) >= 4096:   # token counts change from call to call
            _token_plans.clear()
        _token_plans[key] = p
    return p


def _dense(t):
    """`t` as the kernels address it: contiguous, from a 16-byte boundary on."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _same_device(name, first, *others):
    index = first.get_device()      # (-1: the host's memory)
    for t in others:
        if t is not None and not _is_tensor(t):
            raise RockError("%s: %r is not a tensor" % (name, t))
        if t is not None and t.get_device() != index:
            raise RockError("%s: a tensor is on %s, the first operand on %s" % (name, t.device, first.device))


def _elsewhere(device, stream):
    """The call is for another stream or device than the current ones."""
    return stream is not None or (device.type == "cuda" and device.index != torch._C._cuda_getDevice())


def _on(name, device, stream):
    """A context that makes the operands' device the current one and `stream` (default: the device's current stream)
    torch's current stream, so that copies and results made on the way are ordered with the kernels."""
    if device.type != "cuda":
        return contextlib.ExitStack()
    with contextlib.ExitStack() as stack:      # (left by an exception, it puts the device back)
        stack.enter_context(torch.cuda.device(device))
        if stream is not None:
            if not isinstance(stream, torch.cuda.Stream):
                try:
                    handle = int(getattr(stream, "cuda_stream", stream))
                except (TypeError, ValueError):
                    raise RockError("%s: %r is no stream" % (name, stream))
                # (handle 0 is the default stream; ExternalStream(0) would be one of torch's own, ordered with nothing)
                stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
            if stream.device != device:
                raise RockError("%s: the stream is on %s, the tensors on %s" % (name, stream.device, device))
            stack.enter_context(torch.cuda.stream(stream))
        return stack.pop_all()


def _depth_of_one(rows, weights, axis):
    """Operands of a product over no depth as ones of depth 1 (`axis` of the weights) that hold zeros: the same sums."""
    shape = list(weights.shape)
    shape[axis] = 1
    return rows.new_zeros(rows.shape[:-1] + (1,)), weights.new_zeros(shape)


def _result(name, out, shape, dtype, like, *operands):
    """`out` checked, or a new tensor on `like`'s device.  `operands`: whatever else the call reads or writes."""
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    begin, end = out.data_ptr(), out.data_ptr() + out.nbytes
    for t in (like,) + operands:
        if t is None:
            continue
        span = t.nbytes   # with strides: from the first to the last element
        if not t.is_contiguous() and span:
            span = (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()
        if begin < t.data_ptr() + span and t.data_ptr() < end:
            raise RockError("%s: a result overlaps an operand or another result" % name)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != like.device:
        raise RockError("%s: out must be %s of %s on %s" % (name, tuple(shape), dtype, like.device))
    if not out.is_contiguous() or out.data_ptr() & 15:
        raise RockError("%s: out must be contiguous and start on a 16-byte boundary" % name)
    return out


def _launch_tokens(prog, info, *tensors):
    if info is not None:
        info["kernels"] = [k.kernel_name for k in prog.kernels]
        info["kernel_name"] = prog.kernel_name
        info["perf_config"] = prog.perf_config
    with prog.lock:
        prog.kernels[0].launch_checked(tensors)   # (these problems have one kernel)


def _scale_vector(name, what, t, count):
    if not _is_tensor(t) or t.dtype != torch.float32 or t.numel() != count:
        raise RockError("%s: %s must hold %d float32 elements" % (name, what, count))
    return _dense(t)


def quantize_tokens(x, *, out=None, scale_out=None, stream=None, info=None):
    """Quantises every row of x [..., K] (f16, bf16 or f32) to int8 with a scale of its own, the operands of gemm()
    and grouped_gemm() with `token_scale`: scale = max |x| / 127, q = roundeven(127 x / max |x|).  A row of zeros has
    scale 0 and q = 0; a row that holds an infinity or a NaN has scale NaN and q = 0, so that products of this row,
    and of no other, are NaN.  Returns (q [..., K] int8, scale [...] float32), written into `out` and `scale_out`
    where given."""
    if torch is None:
        _load_torch()
    name = "quantize_tokens"
    shape = x.shape
    if not shape or x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise RockError("quantize_tokens: x is [..., K] of f16, bf16 or f32")
    if _elsewhere(x.device, stream):
        with _on(name, x.device, stream):
            return quantize_tokens(x, out=out, scale_out=scale_out, info=info)
    q = _result(name, out, shape, torch.int8, x)
    s = _result(name, scale_out, shape[:-1], torch.float32, x, q)
    count, cols = x.numel(), shape[-1]
    if count == 0:
        return q, s.zero_()   # rows without elements: their largest magnitude is 0
    _launch_tokens(_token_plan("operation t m k", name, _dtype_name(x.dtype), count // cols, cols), info, _dense(x), q, s)
    return q, s


def _token_scaled_gemm(a, b, transB, out_dtype, scale, zero_point, bias, relu, activation, clip, out, perf_config, stream,
                       info, token_scale):
    """gemm() with a scale for each row of the result."""
    if torch is None:
        _load_torch()
    name = "gemm with token_scale"
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise RockError("%s: int8 operands" % name)
    if a.dim() not in (2, 3) or b.dim() not in (2, 3) or (a.dim() == 3 and a.shape[0] != 1) or (b.dim() == 3 and b.shape[0] != 1):
        raise RockError("%s: one batch entry" % name)
    M, K = a.shape[-2:]
    Kb, N = (b.shape[-1], b.shape[-2]) if transB else (b.shape[-2], b.shape[-1])
    if Kb != K:
        raise RockError("%s: operand shapes do not match" % name)
    if activation not in (None, "relu", "clip") or (activation == "clip" and clip is None):
        raise RockError("%s: activations relu and clip only" % name)
    out_dtype = out_dtype or "f16"
    if out_dtype not in ("f16", "bf16", "f32"):
        raise RockError("%s: out_dtype f16, bf16 or f32" % name)
    vector = _is_tensor(scale)
    _same_device(name, a, b, token_scale, scale if vector else None, bias)
    if _elsewhere(a.device, stream):
        with _on(name, a.device, stream):
            return _token_scaled_gemm(a, b, transB, out_dtype, scale, zero_point, bias, relu, activation, clip, out,
                                      perf_config, None, info, token_scale)
    tensors = [_dense(a), _dense(b), None, None if bias is None else _scale_vector(name, "bias", bias, N),
               _scale_vector(name, "token_scale", token_scale, M)]
    if vector:
        tensors.append(_scale_vector(name, "scale", scale, N))
    res = tensors[2] = _result(name, out, (M, N) if a.dim() == 2 else (1, M, N), _torch_dtype(out_dtype), a, b, token_scale,
                               scale if vector else None, bias)
    if M == 0 or N == 0:
        return res
    if K == 0:
        K = 1
        tensors[0], tensors[1] = _depth_of_one(a, b, -1 if transB else -2)
    lo, hi = (None, None) if clip is None else (float(clip[0]), float(clip[1]))
    prog = _token_plan("operation t token_scale_vector m n k transB out_datatype scale_vector scale zero_point bias "
                       "activation clip_min clip_max perf_config", "gemm", "i8", True, M, N, K, bool(transB), out_dtype,
                       vector, None if vector or scale is None else float(scale), int(zero_point) or None,
                       bias is not None, "clip" if clip is not None else "relu" if relu else activation, lo, hi,
                       perf_config)
    _launch_tokens(prog, info, *tensors)
    return res


def _check_offsets(name, offsets, E):
    if E < 1:
        raise RockError("%s: no experts" % name)
    if not _is_tensor(offsets) or offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] != E + 1:
        raise RockError("%s: offsets is int32 [E + 1], the first row of every expert and the end of the last" % name)


def _grouped(name, rows, w, offsets, transB, cols_of_rows):
    """(groups, rows, N, K) of a grouped product, its operands checked; `cols_of_rows`: what `rows` holds per row."""
    if w.dim() != 3 or rows.dim() != 2 or rows.dtype != w.dtype:
        raise RockError("%s: rows [T, .] and weights [E, ., .] of one type" % name)
    E = w.shape[0]
    N, K = (w.shape[1], w.shape[2]) if transB else (w.shape[2], w.shape[1])
    if rows.shape[1] != (K if cols_of_rows == "K" else N):
        raise RockError("%s: operand shapes do not match" % name)
    _check_offsets(name, offsets, E)
    return E, rows.shape[0], N, K


def grouped_gemm(x, w, offsets, *, transB=False, out_dtype=None, token_scale=None, scale=None, out=None, stream=None,
                 perf_config=None, info=None):
    """Products grouped by expert: rows offsets[e] <= t < offsets[e + 1] of x [T, K] times w[e], w [E, K, N]
    ([E, N, K] if transB) -> [T, N].  `offsets` is int32 [E + 1] on the GPU, never read on the host: non-decreasing
    values within [0, T] (one below 0 is taken as 0, one beyond T as T, one that steps back as the furthest one before
    it).  Experts may have no rows, K may be 0 (sums of nothing are 0); rows of no expert are not written: they keep
    what `out` held (undefined without `out`).  f16, bf16 and f32 operands give a result of their type unless
    `out_dtype` names another of the three; int8 operands give sum * scale * token_scale as f16 (default), bf16 or f32,
    `token_scale` float32 [T], `scale` float32 [E, N] or a number (both optional)."""
    if torch is None:
        _load_torch()
    name = "grouped_gemm"
    E, T, N, K = _grouped(name, x, w, offsets, transB, "K")
    i8 = x.dtype == torch.int8
    t = _dtype_name(x.dtype)
    if t not in ("f32", "f16", "bf16", "i8"):
        raise RockError("%s: f16, bf16, f32 or int8 operands" % name)
    if not i8 and (token_scale is not None or scale is not None):
        raise RockError("%s: scales go with int8 operands" % name)
    out_dtype = out_dtype or ("f16" if i8 else t)
    if out_dtype not in ("f16", "bf16", "f32"):
        raise RockError("%s: out_dtype f16, bf16 or f32" % name)
    vector = _is_tensor(scale)
    _same_device(name, x, w, offsets, token_scale, scale if vector else None)
    if _elsewhere(x.device, stream):
        with _on(name, x.device, stream):
            return grouped_gemm(x, w, offsets, transB=transB, out_dtype=out_dtype, token_scale=token_scale, scale=scale,
                                out=out, perf_config=perf_config, info=info)
    tensors = [_dense(x), _dense(w), None, _dense(offsets)]
    if token_scale is not None:
        tensors.append(_scale_vector(name, "token_scale", token_scale, T))
    if vector:
        tensors.append(_scale_vector(name, "scale", scale, E * N))
        if scale.dim() > 1 and [d for d in scale.shape if d != 1] != [d for d in (E, N) if d != 1]:
            raise RockError("%s: scale is [E, N], not %s" % (name, list(scale.shape)))
    res = tensors[2] = _result(name, out, (T, N), _torch_dtype(out_dtype), x, w, offsets, token_scale,
                               scale if vector else None)
    if T == 0 or N == 0:
        return res
    if K == 0:
        K = 1
        tensors[0], tensors[1] = _depth_of_one(x, w, 2 if transB else 1)
    prog = _token_plan("operation t g m n k transB out_datatype token_scale_vector scale_vector scale perf_config", name, t,
                       E, T, N, K, bool(transB), out_dtype, token_scale is not None, vector,
                       None if vector or scale is None else float(scale), perf_config)
    _launch_tokens(prog, info, *tensors)
    return res


def grouped_gemm_bwd_data(dout, w, offsets, *, transB=False, out=None, stream=None, perf_config=None, info=None):
    """Gradient of grouped_gemm() with respect to x: rows of `dout` [T, N] times the transpose of their expert's
    weights (w and transB as given to grouped_gemm) -> [T, K] of dout's type, f16, bf16 or f32.  Rows of no expert
    are not written."""
    if torch is None:
        _load_torch()
    name = "grouped_gemm_bwd_data"
    E, T, N, K = _grouped(name, dout, w, offsets, transB, "N")
    t = _dtype_name(dout.dtype)
    if t not in ("f32", "f16", "bf16"):
        raise RockError("%s: f16, bf16 or f32 operands" % name)
    _same_device(name, dout, w, offsets)
    if _elsewhere(dout.device, stream):
        with _on(name, dout.device, stream):
            return grouped_gemm_bwd_data(dout, w, offsets, transB=transB, out=out, perf_config=perf_config, info=info)
    res = _result(name, out, (T, K), dout.dtype, dout, w, offsets)
    if T == 0 or K == 0:
        return res
    if N == 0:
        N = 1
        dout, w = _depth_of_one(dout, w, 1 if transB else 2)
    prog = _token_plan("operation t g m n k transB perf_config", name, t, E, T, N, K, bool(transB), perf_config)
    _launch_tokens(prog, info, res, _dense(w), _dense(dout), _dense(offsets))
    return res


def grouped_gemm_bwd_weight(x, dout, offsets, *, transB=False, out=None, stream=None, perf_config=None, info=None):
    """Gradient of grouped_gemm() with respect to w: for every expert the sum over its rows of x [T, K] and dout
    [T, N] -> [E, K, N] ([E, N, K] if transB) of their type, f16, bf16 or f32, summed in f32.  An expert without rows
    gets zeros."""
    if torch is None:
        _load_torch()
    name = "grouped_gemm_bwd_weight"
    if x.dim() != 2 or dout.dim() != 2 or x.shape[0] != dout.shape[0] or x.dtype != dout.dtype:
        raise RockError("%s: x [T, K] and dout [T, N] of one type" % name)
    E = offsets.shape[0] - 1 if _is_tensor(offsets) and offsets.dim() == 1 else 1   # (anything else is refused below)
    T, K, N = x.shape[0], x.shape[1], dout.shape[1]
    _check_offsets(name, offsets, E)
    t = _dtype_name(x.dtype)
    if t not in ("f32", "f16", "bf16"):
        raise RockError("%s: f16, bf16 or f32 operands" % name)
    _same_device(name, x, dout, offsets)
    if _elsewhere(x.device, stream):
        with _on(name, x.device, stream):
            return grouped_gemm_bwd_weight(x, dout, offsets, transB=transB, out=out, perf_config=perf_config, info=info)
    res = _result(name, out, (E, N, K) if transB else (E, K, N), x.dtype, x, dout, offsets)
    if res.numel() == 0:
        return res
    if T == 0:
        return res.zero_()
    prog = _token_plan("operation t g m n k transB perf_config", name, t, E, T, N, K, bool(transB), perf_config)
    _launch_tokens(prog, info, _dense(x), res, _dense(dout), _dense(offsets))
    return res
