"""ctypes binding of libhat.so (include/hat.h) for the tests and the benchmark.

The product is the C ABI; this module only marshals numpy arrays across it.
It mirrors the reference's host interface: `Weights.load` (src/weights.rs:60),
`Backend.name` / `Backend.forward` (src/backend.rs:29-36), `verify`
(src/main.rs:312-326) and `selftest` (src/selftest.rs:437-523).

There is no CPU fallback: `Backend("gpu")` fails loudly when the library or a
device is missing.
"""
import ctypes as C
import os
import struct

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "build", "libhat.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "hat.h")

_f32p = C.POINTER(C.c_float)


class HatError(RuntimeError):
    pass


class ModelInfo(C.Structure):
    _fields_ = [("scale", C.c_int), ("window", C.c_int), ("owin", C.c_int), ("embed", C.c_int),
                ("heads", C.c_int), ("head_dim", C.c_int), ("mlp_ratio", C.c_int),
                ("n_stages", C.c_int), ("depths", C.c_int * 32), ("compressed", C.c_int),
                ("squeezed", C.c_int), ("head_feat", C.c_int), ("conv_scale", C.c_float),
                ("img_range", C.c_float), ("mean", C.c_float * 3)]


class Tiling(C.Structure):
    _fields_ = [(n, C.c_size_t) for n in ("tile", "margin", "scale", "tiles", "largest_h", "largest_w")]


class Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("batch_stride", C.c_longlong), ("token_stride", C.c_longlong),
                ("head_stride", C.c_longlong)]


class Positions(C.Structure):
    _fields_ = [("data", C.c_void_p), ("batch_stride", C.c_longlong), ("token_stride", C.c_longlong),
                ("axis_stride", C.c_longlong)]


class RotaryArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("batch", C.c_int), ("q_heads", C.c_int), ("k_heads", C.c_int),
                ("head_dim", C.c_int), ("axes", C.c_int), ("tokens", C.c_longlong), ("sections", C.c_int * 4),
                ("joint", C.c_int), ("neighbours", C.c_int), ("inverse", C.c_int), ("base", C.c_double),
                ("pos", Positions), ("q", Heads), ("q_out", Heads), ("k", Heads), ("k_out", Heads)]


class AttentionArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("n_seq", C.c_int), ("q_heads", C.c_int), ("kv_heads", C.c_int),
                ("head_dim", C.c_int), ("axes", C.c_int), ("q_tokens", C.c_longlong), ("k_tokens", C.c_longlong),
                ("q", Heads), ("k", Heads), ("v", Heads), ("out", Heads),
                ("cu_q", C.c_void_p), ("cu_k", C.c_void_p), ("q_lens", C.c_void_p), ("k_lens", C.c_void_p),
                ("prefix", C.c_void_p), ("causal", C.c_int), ("scale", C.c_float), ("cap", C.c_float),
                ("slopes", C.c_void_p), ("pos_q", Positions), ("pos_k", Positions), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class ResidualNormArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("width", C.c_int), ("post", C.c_int), ("pre", C.c_int),
                ("rows", C.c_longlong), ("rows_per_gate", C.c_longlong), ("x", C.c_void_p), ("y", C.c_void_p),
                ("gate", C.c_void_p), ("x_out", C.c_void_p), ("h", C.c_void_p), ("x_stride", C.c_longlong),
                ("y_stride", C.c_longlong), ("gate_stride", C.c_longlong), ("x_out_stride", C.c_longlong),
                ("h_stride", C.c_longlong), ("post_w", C.c_void_p), ("post_b", C.c_void_p), ("pre_w", C.c_void_p),
                ("pre_b", C.c_void_p), ("scale", C.c_float), ("post_eps", C.c_float), ("pre_eps", C.c_float)]


class MemPlan(C.Structure):
    _fields_ = [(n, C.c_ulonglong) for n in ("activations", "weights", "base", "need", "avail")] + \
               [("have_avail", C.c_int)]


_lib = None


def lib():
    """Load libhat.so (built by __graft_entry__.build / `make -C hat-rs_amd`)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise HatError(f"{LIB_PATH} is missing: build it with `make -C hat-rs_amd`")
    L = C.CDLL(LIB_PATH)
    sig = {
        "hat_version": (C.c_char_p, []),
        "hat_last_error": (C.c_char_p, []),
        "hat_weights_open": (C.c_void_p, [C.c_char_p]),
        "hat_weights_close": (None, [C.c_void_p]),
        "hat_weights_info": (C.c_int, [C.c_void_p, C.POINTER(ModelInfo)]),
        "hat_weights_count": (C.c_int, [C.c_void_p]),
        "hat_weights_name": (C.c_char_p, [C.c_void_p, C.c_int]),
        "hat_weights_tensor": (_f32p, [C.c_void_p, C.c_char_p, C.POINTER(C.c_size_t)]),
        "hat_weights_index_i64": (C.c_long, [C.c_void_p, C.c_char_p, C.POINTER(C.c_longlong), C.c_size_t]),
        "hat_weights_generate": (C.c_int, [C.c_char_p, C.c_char_p, C.c_int, C.c_ulonglong,
                                           C.POINTER(C.c_int), C.c_int]),
        "hat_weights_variant": (C.c_char_p, [C.c_void_p]),
        "hat_weights_file_bytes": (C.c_ulonglong, [C.c_void_p]),
        "hat_weights_shape": (C.c_int, [C.c_void_p, C.c_char_p, C.POINTER(C.c_size_t), C.c_int]),
        "hat_backend_forward_batch": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, C.c_size_t, _f32p, _f32p]),
        "hat_tile_forward": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, _f32p, _f32p, C.c_size_t, C.c_size_t,
                                       C.POINTER(Tiling)]),
        "hat_auto_tile": (C.c_size_t, [C.c_size_t, C.c_size_t, C.c_size_t, C.c_ulonglong, C.c_ulonglong,
                                       C.c_ulonglong, C.c_size_t]),
        "hat_gpu_plan": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, C.POINTER(MemPlan)]),
        "hat_gpu_auto_tile": (C.c_long, [C.c_void_p, C.c_size_t, C.c_size_t]),
        "hat_png_load": (C.c_int, [C.c_char_p, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t), _f32p, C.c_size_t]),
        "hat_png_save": (C.c_int, [C.c_char_p, C.c_size_t, C.c_size_t, _f32p]),
        "hat_gpu_available": (C.c_int, []),
        "hat_backend_new": (C.c_void_p, [C.c_void_p, C.c_char_p]),
        "hat_backend_name": (C.c_char_p, [C.c_void_p]),
        "hat_backend_forward": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, _f32p, _f32p]),
        "hat_backend_forward_device": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, C.c_void_p,
                                                 C.c_void_p]),
        "hat_backend_synchronize": (C.c_int, [C.c_void_p]),
        "hat_backend_forward_noalloc": (C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, C.c_void_p,
                                                  C.c_void_p]),
        "hat_backend_hab": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_size_t, C.c_size_t, _f32p, _f32p,
                                      C.c_int, _f32p]),
        "hat_backend_acts_bytes": (C.c_size_t, [C.c_void_p]),
        "hat_backend_weight_bytes": (C.c_size_t, [C.c_void_p]),
        "hat_backend_free": (None, [C.c_void_p]),
        "hat_verify": (C.c_int, [C.c_void_p, C.c_char_p, C.c_char_p]),
        "hat_gpu_selftest": (C.c_int, []),
        "hat_op_swmsa": (C.c_int, [_f32p, _f32p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                   _f32p, _f32p, _f32p, _f32p, _f32p, C.c_int, _f32p, _f32p]),
        "hat_op_ocab": (C.c_int, [_f32p, _f32p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]
                        + [_f32p] * 13 + [C.c_int, _f32p, _f32p]),
        # structures: by reference, or packed bytes
        "hat_op_rotary": (C.c_int, [C.c_void_p, C.c_void_p]),
        "hat_op_attention_workspace": (C.c_size_t, [C.c_void_p]),
        "hat_op_attention": (C.c_int, [C.c_void_p, C.c_void_p]),
        "hat_op_residual_norm": (C.c_int, [C.c_void_p, C.c_void_p]),
        "hat_device_alloc": (C.c_void_p, [C.c_size_t]),
        "hat_device_free": (C.c_int, [C.c_void_p]),
        "hat_memcpy_h2d": (C.c_int, [C.c_void_p, C.c_void_p, C.c_size_t]),
        "hat_memcpy_d2h": (C.c_int, [C.c_void_p, C.c_void_p, C.c_size_t]),
        "hat_device_copy": (C.c_int, [C.c_void_p, C.c_void_p, C.c_size_t]),
        "hat_device_synchronize": (C.c_int, []),
        "hat_device_mem_info": (C.c_int, [C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]),
        "hat_device_name": (C.c_char_p, []),
        "hat_device_cu_count": (C.c_int, []),
        "hat_profile_begin": (C.c_int, []),
        "hat_profile_end": (C.c_int, []),
        "hat_profile_count": (C.c_int, []),
        "hat_profile_get": (C.c_int, [C.c_int, C.c_char_p, C.c_int, C.POINTER(C.c_long),
                                      C.POINTER(C.c_double)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def _err():
    # messages can quote names read from a file: never fail on their bytes
    return lib().hat_last_error().decode(errors="replace")


def _check(rc, what):
    if rc is None or (isinstance(rc, int) and rc < 0):
        raise HatError(f"{what}: {_err()}")
    return rc


def _fp(a):
    return a.ctypes.data_as(_f32p) if a is not None else None


def f32(a):
    return np.ascontiguousarray(a, dtype=np.float32)


def declared_symbols():
    """Every function name include/hat.h declares."""
    import re
    src = open(HEADER).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(hat_[a-z0-9_]+)\s*\(", src)))


# ---------------------------------------------------------------------------

def generate_weights(path, variant="hat-s", scale=4, seed=0, depths=None):
    d = None
    n = 0
    if depths is not None:
        n = len(depths)
        d = (C.c_int * n)(*depths)
    _check(lib().hat_weights_generate(str(path).encode(), variant.encode(), scale, seed, d, n),
           "hat_weights_generate")
    return path


class Weights:
    """Weights::load (src/weights.rs:60)."""

    def __init__(self, path):
        self.path = str(path)
        h = lib().hat_weights_open(self.path.encode())
        if not h:
            raise HatError(_err())
        self.h = h
        info = ModelInfo()
        _check(lib().hat_weights_info(h, C.byref(info)), "hat_weights_info")
        self.info = info
        self.scale = info.scale
        self.window = info.window
        self.owin = info.owin
        self.embed = info.embed
        self.heads = info.heads
        self.head_dim = info.head_dim
        self.mlp_ratio = info.mlp_ratio
        self.depths = [info.depths[i] for i in range(info.n_stages)]
        self.compressed = info.compressed
        self.squeezed = info.squeezed
        self.head_feat = info.head_feat
        self.conv_scale = info.conv_scale
        self.img_range = info.img_range
        self.mean = [info.mean[i] for i in range(3)]

    def variant(self):
        return lib().hat_weights_variant(self.h).decode()

    def file_bytes(self):
        return lib().hat_weights_file_bytes(self.h)

    def shape(self, name):
        d = (C.c_size_t * 16)()
        n = _check(lib().hat_weights_shape(self.h, name.encode(), d, 16), "hat_weights_shape")
        return [d[i] for i in range(n)]

    def gpu_plan(self, h, w):
        p = MemPlan()
        _check(lib().hat_gpu_plan(self.h, h, w, C.byref(p)), "hat_gpu_plan")
        return {n: getattr(p, n) for n, _ in MemPlan._fields_}

    def names(self):
        L = lib()
        return [L.hat_weights_name(self.h, i).decode() for i in range(L.hat_weights_count(self.h))]

    def tensor(self, name):
        n = C.c_size_t(0)
        p = lib().hat_weights_tensor(self.h, name.encode(), C.byref(n))
        if not p:
            raise HatError(_err())
        return np.ctypeslib.as_array(p, shape=(n.value,))

    def i64(self, name):
        L = lib()
        n = L.hat_weights_index_i64(self.h, name.encode(), None, 0)
        _check(n, "hat_weights_index_i64")
        out = np.zeros(n, dtype=np.int64)
        L.hat_weights_index_i64(self.h, name.encode(), out.ctypes.data_as(C.POINTER(C.c_longlong)), n)
        return out

    def close(self):
        if self.h:
            lib().hat_weights_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def gpu_available():
    return bool(lib().hat_gpu_available())


class Backend:
    """The MI355X backend behind the reference's `Backend` trait (src/backend.rs:29-36)."""

    def __init__(self, weights, device="gpu"):
        self.weights = weights
        h = lib().hat_backend_new(weights.h, device.encode())
        if not h:
            raise HatError(_err())
        self.h = h

    def name(self):
        return lib().hat_backend_name(self.h).decode()

    def forward(self, h, w, img, out=None):
        """Backend::forward; `out` (optional) is a caller-allocated
        [3][h*s][w*s] float32 array, as the C ABI's output argument is."""
        img = f32(img).reshape(3, h, w)
        s = self.weights.scale
        if out is None:
            out = np.empty((3, h * s, w * s), dtype=np.float32)
        assert out.shape == (3, h * s, w * s) and out.dtype == np.float32 and out.flags["C_CONTIGUOUS"]
        _check(lib().hat_backend_forward(self.h, h, w, _fp(img), _fp(out)), "forward")
        return out

    def forward_device(self, h, w, d_in, d_out):
        _check(lib().hat_backend_forward_device(self.h, h, w, d_in, d_out), "forward_device")

    def forward_batch(self, n, h, w, imgs):
        imgs = f32(imgs).reshape(n, 3, h, w)
        s = self.weights.scale
        out = np.empty((n, 3, h * s, w * s), dtype=np.float32)
        _check(lib().hat_backend_forward_batch(self.h, n, h, w, _fp(imgs), _fp(out)), "forward_batch")
        return out

    def tile_forward(self, h, w, img, tile, margin):
        img = f32(img).reshape(3, h, w)
        s = self.weights.scale
        out = np.empty((3, h * s, w * s), dtype=np.float32)
        t = Tiling()
        _check(lib().hat_tile_forward(self.h, h, w, _fp(img), _fp(out), tile, margin, C.byref(t)),
               "tile_forward")
        return out, {n: getattr(t, n) for n, _ in Tiling._fields_}

    def forward_noalloc(self, h, w, d_in, d_out):
        _check(lib().hat_backend_forward_noalloc(self.h, h, w, d_in, d_out), "forward_noalloc")

    def synchronize(self):
        _check(lib().hat_backend_synchronize(self.h), "synchronize")

    def hab(self, stage, block, hp, wp, x, iters=0):
        """One HAB (gpu.rs:469-520) on a token-major [hp*wp][embed] plane; returns
        (out, mean ms over `iters` further runs)."""
        x = f32(x).reshape(hp * wp, self.weights.embed)
        out = np.empty_like(x)
        ms = C.c_float(0)
        _check(lib().hat_backend_hab(self.h, stage, block, hp, wp, _fp(x), _fp(out), iters,
                                     C.cast(C.byref(ms), _f32p)), "hat_backend_hab")
        return out, ms.value

    def acts_bytes(self):
        return lib().hat_backend_acts_bytes(self.h)

    def weight_bytes(self):
        return lib().hat_backend_weight_bytes(self.h)

    def close(self):
        if self.h:
            lib().hat_backend_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def verify(weights, fixture_path, device="gpu"):
    rc = lib().hat_verify(weights.h, device.encode(), str(fixture_path).encode())
    if rc < 0:
        raise HatError(_err())
    return rc


def auto_tile(h, w, win, budget_bytes, per_pixel_floats, constant_floats, margin):
    """tile::auto_tile; None when not even one window fits."""
    t = lib().hat_auto_tile(h, w, win, budget_bytes, per_pixel_floats, constant_floats, margin)
    return t or None


def png_load(path):
    w, h = C.c_size_t(0), C.c_size_t(0)
    _check(lib().hat_png_load(str(path).encode(), C.byref(w), C.byref(h), None, 0), "hat_png_load")
    out = np.empty((3, h.value, w.value), dtype=np.float32)
    _check(lib().hat_png_load(str(path).encode(), C.byref(w), C.byref(h), _fp(out), out.size), "hat_png_load")
    return out


def png_save(path, planes):
    planes = f32(planes)
    c, h, w = planes.shape
    assert c == 3
    _check(lib().hat_png_save(str(path).encode(), w, h, _fp(planes)), "hat_png_save")


CLI_PATH = os.path.join(HERE, "build", "hat")


def selftest():
    return _check(lib().hat_gpu_selftest(), "selftest")


def op_swmsa(x, hp, wp, c, heads, shift, qkv_w, qkv_b, proj_w, proj_b, table, iters=0):
    x = f32(x)
    out = np.empty_like(x)
    ms = C.c_float(0)
    ams = C.c_float(0)
    args = [f32(a) for a in (qkv_w, qkv_b, proj_w, proj_b, table)]
    _check(lib().hat_op_swmsa(_fp(x), _fp(out), hp, wp, c, heads, shift, *[_fp(a) for a in args],
                              iters, C.cast(C.byref(ms), _f32p), C.cast(C.byref(ams), _f32p)),
           "hat_op_swmsa")
    return out, ms.value, ams.value


def op_ocab(x, hp, wp, c, heads, mlp_ratio, ws, iters=0):
    """ws: the 13 OCAB tensors in the order of include/hat.h."""
    x = f32(x)
    out = np.empty_like(x)
    ms = C.c_float(0)
    ams = C.c_float(0)
    args = [f32(a) for a in ws]
    _check(lib().hat_op_ocab(_fp(x), _fp(out), hp, wp, c, heads, mlp_ratio,
                             *[_fp(a) for a in args], iters, C.cast(C.byref(ms), _f32p),
                             C.cast(C.byref(ams), _f32p)), "hat_op_ocab")
    return out, ms.value, ams.value


class DeviceBuffer:
    def __init__(self, nbytes):
        self.nbytes = nbytes
        self.ptr = lib().hat_device_alloc(nbytes)
        if not self.ptr:
            raise HatError(_err())

    def upload(self, arr):
        arr = np.ascontiguousarray(arr)
        assert arr.nbytes <= self.nbytes
        _check(lib().hat_memcpy_h2d(self.ptr, arr.ctypes.data, arr.nbytes), "h2d")

    def download(self, arr):
        assert arr.nbytes <= self.nbytes and arr.flags["C_CONTIGUOUS"]
        _check(lib().hat_memcpy_d2h(arr.ctypes.data, self.ptr, arr.nbytes), "d2h")
        return arr

    def free(self):
        if self.ptr:
            lib().hat_device_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def synchronize():
    _check(lib().hat_device_synchronize(), "synchronize")


def device_copy(dst, src, nbytes):
    """Device-to-device copy with the library's copy kernel (DeviceBuffer or raw pointers)."""
    d = dst.ptr if isinstance(dst, DeviceBuffer) else dst
    s = src.ptr if isinstance(src, DeviceBuffer) else src
    _check(lib().hat_device_copy(d, s, nbytes), "device_copy")


def device_mem_info():
    """(free, total) device memory in bytes."""
    fr, tot = C.c_size_t(0), C.c_size_t(0)
    _check(lib().hat_device_mem_info(C.byref(fr), C.byref(tot)), "device_mem_info")
    return fr.value, tot.value


def device_name():
    return lib().hat_device_name().decode()


def device_cu_count():
    return lib().hat_device_cu_count()


def profile_begin():
    _check(lib().hat_profile_begin(), "profile_begin")


def profile_end():
    """Stop timing; return {kernel: (launches, total_ms)}."""
    L = lib()
    _check(L.hat_profile_end(), "profile_end")
    out = {}
    buf = C.create_string_buffer(128)
    for i in range(L.hat_profile_count()):
        cnt = C.c_long(0)
        tot = C.c_double(0)
        _check(L.hat_profile_get(i, buf, 128, C.byref(cnt), C.byref(tot)), "profile_get")
        out[buf.value.decode()] = (cnt.value, tot.value)
    return out


# ---------------------------------------------------------------------------
# Operators on device tensors (include/hat.h). A device tensor is a DeviceArray or any
# object with its five methods and attributes: data_ptr(), get_device() (0: the
# library's device), stride() in elements, shape and dtype, as torch's tensors have.

_DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "int32": 3, "uint8": 4}
_SIZES = {0: 4, 1: 2, 2: 2, 3: 4, 4: 1}
_NORMS = {"none": 0, "layer": 1, "rms": 2}
_dtype_codes = {}


class DeviceArray:
    """A contiguous device tensor of its own: a DeviceBuffer with a shape and a type
    ("float32", "float16", "bfloat16", "int32", "uint8")."""

    def __init__(self, shape, dtype, data=None):
        self.shape, self.dtype = tuple(shape), dtype
        count = 1
        for n in self.shape:
            count *= n
        self.buffer = DeviceBuffer(max(4, count * _SIZES[_DTYPES[dtype]]))
        if data is not None:
            data = np.ascontiguousarray(data)
            if data.nbytes != count * _SIZES[_DTYPES[dtype]]:
                raise HatError(f"DeviceArray: {data.nbytes} bytes for a shape of {self.shape} in {dtype}")
            if data.nbytes:
                self.buffer.upload(data)

    def data_ptr(self):
        return self.buffer.ptr

    def get_device(self):
        return 0

    def stride(self):
        s, out = 1, []
        for n in reversed(self.shape):
            out.append(s)
            s *= n
        return tuple(reversed(out))

    def numpy(self):
        """A copy on the host; bfloat16 as its uint16 bits."""
        kind = {"bfloat16": "uint16"}.get(self.dtype, self.dtype)
        out = np.empty(self.shape, dtype=kind)
        return self.buffer.download(out) if out.nbytes else out


def _code(t, what):
    """The type of a device tensor as the C ABI's number; refuses what is not on the device."""
    d = t.dtype
    c = _dtype_codes.get(d)
    if c is None:
        c = _DTYPES.get(str(d).replace("torch.", ""))
        if c is None:
            raise HatError(f"{what}: type {d} is not supported")
        _dtype_codes[d] = c
    if t.get_device() != 0:
        raise HatError(f"{what}: not a tensor of device 0")
    return c


_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(lib(), name)
    return f


def _packed(op, layout, *fields):
    try:
        return layout.pack(*fields)
    except (struct.error, OverflowError) as e:  # a size or a factor that its field cannot hold
        raise HatError(f"{op}: an argument is out of range ({e})")


# The argument structures packed in one go, field by field as they are declared above
# (a ctypes structure costs a call an assignment a field).
_ROTARY = struct.Struct("@6iq4i3id4q16q")
_ATTENTION = struct.Struct("@6i2q16q5QifffQ8qQQ")
_NORM = struct.Struct("@4i2q5Q5q4Q3f4x")
_NO_HEADS = (0, 0, 0, 0)


def _heads(t, what, code, lead=None):
    """(the fields of Heads, batch, tokens, heads, dim) of [batch, token, head, dim] or
    [token, head, dim]."""
    if _code(t, what) != code:
        raise HatError(f"{what}: type {t.dtype} differs from the first tensor's")
    shape, st = t.shape, t.stride()
    if lead is not None and shape != lead:
        raise HatError(f"{what}: {tuple(shape)} where {tuple(lead)} is expected")
    n = len(shape)
    if n == 4:
        batch, tokens, heads, dim = shape
        fields = (t.data_ptr(), st[0], st[1], st[2])
    elif n == 3:
        tokens, heads, dim = shape
        batch, fields = 1, (t.data_ptr(), 0, st[0], st[1])
    else:
        raise HatError(f"{what}: [batch, token, head, dim] or [token, head, dim] expected, not {tuple(shape)}")
    if st[-1] != 1 and dim > 1:
        raise HatError(f"{what}: the last axis must have stride 1")
    return fields, batch, tokens, heads, dim


def _positions(t, what, batch, tokens):
    """(the fields of Positions, axes) of int32 [token, axis], shared by the batch, or
    [batch, token, axis]."""
    if _code(t, what) != 3:
        raise HatError(f"{what}: int32 expected, not {t.dtype}")
    shape, st = t.shape, t.stride()
    if len(shape) == 2 and shape[0] == tokens:
        return (t.data_ptr(), 0, st[0], st[1]), shape[1]
    if len(shape) == 3 and shape[0] == batch and shape[1] == tokens:
        return (t.data_ptr(), st[0], st[1], st[2]), shape[2]
    raise HatError(f"{what}: {tuple(shape)} is no [{tokens}, axis] or [{batch}, {tokens}, axis]")


def _vector(t, what, code, n):
    """The pointer of a contiguous vector of n values, or 0."""
    if t is None:
        return 0
    shape = t.shape
    if _code(t, what) != code or len(shape) != 1 or shape[0] != n or (n > 1 and t.stride()[0] != 1):
        raise HatError(f"{what}: {n} contiguous values of {'fp32' if code == 0 else 'int32'} expected")
    return t.data_ptr()


def op_rotary(q, k, pos, sections, base=10000.0, pairs="halves", joint=False, inverse=False, q_out=None, k_out=None,
              stream=None):
    """hat_op_rotary: turns q and k (None: q alone) by their tokens' positions, in place
    where q_out / k_out are left out. pairs: "halves" or "neighbours"; stream: a
    hipStream_t as an integer (torch's `cuda_stream`), None the default stream."""
    code = _code(q, "rotary: q")
    fq, batch, tokens, q_heads, dim = _heads(q, "rotary: q", code)
    fqo = fq if q_out is None else _heads(q_out, "rotary: q_out", code, q.shape)[0]
    k_heads, fk, fko = 0, _NO_HEADS, _NO_HEADS
    if k is not None:
        fk, b, t, k_heads, d = _heads(k, "rotary: k", code)
        if b != batch or t != tokens or d != dim:
            raise HatError(f"rotary: k of {tuple(k.shape)} does not go with q of {tuple(q.shape)}")
        fko = fk if k_out is None else _heads(k_out, "rotary: k_out", code, k.shape)[0]
    elif k_out is not None:
        raise HatError("rotary: k_out without k")
    fp, axes = _positions(pos, "rotary: pos", batch, tokens)
    if axes != len(sections) or not 1 <= axes <= 4:
        raise HatError(f"rotary: {axes} axes of positions and {len(sections)} sections (1 to 4)")
    if pairs not in ("halves", "neighbours"):
        raise HatError(f"rotary: pairs are halves or neighbours, not {pairs!r}")
    _check(_fn("hat_op_rotary")(_packed("rotary", _ROTARY, code, batch, q_heads, k_heads, dim, axes, tokens,
                                        *sections, *(0,) * (4 - axes), bool(joint), pairs == "neighbours",
                                        bool(inverse), base, *fp, *fq, *fqo, *fk, *fko), stream), "rotary")


def _sequences(cu, what):
    if len(cu.shape) != 1 or cu.shape[0] < 1:
        raise HatError(f"{what}: offsets of every sequence and the end of the last expected")
    return cu.shape[0] - 1


def _attention_args(q, k, v, out, scale, causal, prefix, cu_q, cu_k, q_lens, k_lens, cap, slopes, pos_q, pos_k,
                    workspace=0, workspace_bytes=0):
    code = _code(q, "attention: q")
    fq, bq, q_tokens, q_heads, dim = _heads(q, "attention: q", code)
    fk, bk, k_tokens, kv_heads, d = _heads(k, "attention: k", code)
    fv = _heads(v, "attention: v", code, k.shape)[0]
    fo = _heads(out, "attention: out", code, q.shape)[0]
    if d != dim:
        raise HatError(f"attention: head_dim {dim} of q and {d} of k")
    n = bq
    if cu_q is not None or cu_k is not None:
        n = _sequences(cu_q, "attention: cu_q") if cu_q is not None else None
        if cu_k is not None:
            m = _sequences(cu_k, "attention: cu_k")
            if n is not None and m != n:
                raise HatError(f"attention: {n} sequences in cu_q and {m} in cu_k")
            n = m
        if (cu_q is not None and len(q.shape) != 3) or (cu_k is not None and len(k.shape) != 3):
            raise HatError("attention: a packed tensor is [token, head, dim]")
    if (cu_q is None and bq != n) or (cu_k is None and bk != n):
        raise HatError(f"attention: q of {tuple(q.shape)} and k of {tuple(k.shape)} are not {n} sequences")
    axes, fpq, fpk = 0, _NO_HEADS, _NO_HEADS
    if pos_q is not None and pos_k is not None:
        fpq, axes = _positions(pos_q, "attention: pos_q", bq, q_tokens)
        fpk, d = _positions(pos_k, "attention: pos_k", bk, k_tokens)
        if d != axes:
            raise HatError(f"attention: {axes} axes in pos_q and {d} in pos_k")
    elif pos_q is not None or pos_k is not None:
        raise HatError("attention: positions of queries and keys go together")
    return _packed("attention", _ATTENTION, code, n, q_heads, kv_heads, dim, axes, q_tokens, k_tokens, *fq, *fk, *fv,
                   *fo, _vector(cu_q, "attention: cu_q", 3, n + 1), _vector(cu_k, "attention: cu_k", 3, n + 1),
                   _vector(q_lens, "attention: q_lens", 3, n), _vector(k_lens, "attention: k_lens", 3, n),
                   _vector(prefix, "attention: prefix", 3, n), bool(causal), dim ** -0.5 if scale is None else scale,
                   cap, 0.0, _vector(slopes, "attention: slopes", 0, q_heads), *fpq, *fpk, workspace, workspace_bytes)


def attention_workspace(q, k, v, out, scale=None, causal=False, prefix=None, cu_q=None, cu_k=None, q_lens=None,
                        k_lens=None, cap=0.0, slopes=None, pos_q=None, pos_k=None):
    """The bytes that op_attention of these arguments needs as its workspace."""
    n = _fn("hat_op_attention_workspace")(_attention_args(q, k, v, out, scale, causal, prefix, cu_q, cu_k, q_lens,
                                                          k_lens, cap, slopes, pos_q, pos_k))
    if n == C.c_size_t(-1).value:
        raise HatError(f"attention: {_err()}")
    return n


def op_attention(q, k, v, out, scale=None, causal=False, prefix=None, cu_q=None, cu_k=None, q_lens=None, k_lens=None,
                 cap=0.0, slopes=None, pos_q=None, pos_k=None, workspace=None, stream=None):
    """hat_op_attention: [batch, token, head, dim] tensors, or packed [token, head, dim] with
    cu_q / cu_k; scale None: head_dim^-1/2; workspace: a device tensor of at least
    attention_workspace(...) bytes where that is not 0; stream as op_rotary's."""
    ptr = size = 0
    if workspace is not None:
        size = _SIZES[_code(workspace, "attention: workspace")]
        if len(workspace.shape) != 1 or (workspace.shape[0] > 1 and workspace.stride()[0] != 1):
            raise HatError("attention: the workspace is one contiguous row")
        ptr, size = workspace.data_ptr(), workspace.shape[0] * size
    _check(_fn("hat_op_attention")(_attention_args(q, k, v, out, scale, causal, prefix, cu_q, cu_k, q_lens, k_lens, cap,
                                                   slopes, pos_q, pos_k, ptr, size), stream), "attention")


def _rows(t, what, code, lead=None):
    """(pointer, row stride) of [rows, width]."""
    if _code(t, what) != code:
        raise HatError(f"{what}: type {t.dtype} differs from x's")
    shape, st = t.shape, t.stride()
    if len(shape) != 2 or (st[1] != 1 and shape[1] > 1) or (lead is not None and shape != lead):
        raise HatError(f"{what}: {tuple(shape)} is no [rows, width] of stride 1" + (f" like x's {tuple(lead)}" if lead else ""))
    return t.data_ptr(), st[0]


def op_residual_norm(x, y=None, x_out=None, h=None, gate=None, scale=1.0, post="none", post_weight=None,
                     post_bias=None, pre="none", pre_weight=None, pre_bias=None, eps=1e-5, post_eps=None,
                     stream=None):
    """hat_op_residual_norm on [rows, width] tensors: x_out = x + scale * gate * N(y), h =
    N(x_out), either left out where None. gate: [gates, width], a row for each rows / gates
    rows; post, pre: "none", "layer" or "rms" with fp32 weights; post_eps None: eps."""
    code = _code(x, "residual_norm: x")
    if code > 2:
        raise HatError(f"residual_norm: type {x.dtype} is not supported")
    px, sx = _rows(x, "residual_norm: x", code)
    lead = x.shape
    rows, width = lead
    py = sy = pxo = sxo = ph = sh = pg = sg = 0
    per = 1
    if y is not None:
        py, sy = _rows(y, "residual_norm: y", code, lead)
    if x_out is not None:
        pxo, sxo = _rows(x_out, "residual_norm: x_out", code, lead)
    if h is not None:
        ph, sh = _rows(h, "residual_norm: h", code, lead)
    if gate is not None:
        pg, sg = _rows(gate, "residual_norm: gate", code)
        n = gate.shape[0]
        if gate.shape[1] != width or n < 1 or rows % n:
            raise HatError(f"residual_norm: gates of {tuple(gate.shape)} for x of {tuple(lead)}")
        per = max(1, rows // n)
    if post not in _NORMS or pre not in _NORMS:
        raise HatError(f"residual_norm: norms are none, layer or rms, not {post!r}, {pre!r}")
    _check(_fn("hat_op_residual_norm")(_packed(
        "residual_norm", _NORM, code, width, _NORMS[post], _NORMS[pre], rows, per, px, py, pg, pxo, ph, sx, sy, sg, sxo, sh,
        _vector(post_weight, "residual_norm: post_weight", 0, width),
        _vector(post_bias, "residual_norm: post_bias", 0, width),
        _vector(pre_weight, "residual_norm: pre_weight", 0, width),
        _vector(pre_bias, "residual_norm: pre_bias", 0, width), scale, eps if post_eps is None else post_eps, eps),
        stream), "residual_norm")
