"""ctypes binding of the C ABI in include/sblocal_b200.h.

The library is loaded from fly_b200/lib (built in-tree by fly_b200.build).
There is no fallback: if the library is missing or a call fails, an exception
is raised.
"""
import ctypes
import os
import struct
import threading

from . import build as _build

SBL_DTYPE_F32 = 0
SBL_DTYPE_BF16 = 1
SBL_FLAG_GENERIC_PATH = 1
SBL_SKIP = (1, 2, 4)   # SBL_SKIP_DQ, SBL_SKIP_DK, SBL_SKIP_DV

SBL_OK = 0
SBL_ERR_INVALID_ARGUMENT = -1
SBL_ERR_UNSUPPORTED = -2
SBL_ERR_WORKSPACE = -3
SBL_ERR_CUDA = -4
SBL_ERR_DEVICE_STATUS = -5

ABI_VERSION = 1

EXPORTS = ('sbl_version', 'sbl_last_error', 'sbl_has_tensor_path', 'sbl_workspace_bytes', 'sbl_forward',
           'sbl_key_logscale', 'sbl_key_summary', 'sbl_band_forward', 'sbl_query_features',
           'sbl_key_features', 'sbl_attention_weights', 'sbl_check_status', 'sbl_selftest_wait_timeout',
           'sbl_key_logscale_static', 'sbl_static_last_error', 'sbl_status_words', 'sbl_forward_train',
           'sbl_backward_workspace_bytes', 'sbl_backward', 'sbl_norm_rotary_forward',
           'sbl_norm_rotary_workspace_bytes', 'sbl_norm_rotary_backward', 'sbl_collect_status')


class SblParams(ctypes.Structure):
    """Mirror of `struct SblParams`."""
    _fields_ = [
        ('dtype', ctypes.c_int32),
        ('B', ctypes.c_int32), ('H', ctypes.c_int32), ('T', ctypes.c_int32), ('S', ctypes.c_int32),
        ('E', ctypes.c_int32), ('D', ctypes.c_int32),
        ('r', ctypes.c_int32),
        ('w', ctypes.c_int32),
        ('softmax_temp', ctypes.c_float),
        ('softmax_eps', ctypes.c_float),
        ('q', ctypes.c_void_p), ('q_stride_b', ctypes.c_int64), ('q_stride_t', ctypes.c_int64),
        ('q_stride_h', ctypes.c_int64),
        ('k', ctypes.c_void_p), ('k_stride_b', ctypes.c_int64), ('k_stride_s', ctypes.c_int64),
        ('k_stride_h', ctypes.c_int64),
        ('v', ctypes.c_void_p), ('v_stride_b', ctypes.c_int64), ('v_stride_s', ctypes.c_int64),
        ('v_stride_h', ctypes.c_int64),
        ('out', ctypes.c_void_p), ('o_stride_b', ctypes.c_int64), ('o_stride_t', ctypes.c_int64),
        ('o_stride_h', ctypes.c_int64),
        ('W', ctypes.c_void_p),
        ('key_lengths', ctypes.c_void_p),
        ('q_pos0', ctypes.c_int64), ('k_pos0', ctypes.c_int64),
        ('S_total', ctypes.c_int64),
        ('sum_lo', ctypes.c_int32), ('sum_hi', ctypes.c_int32),
        ('flags', ctypes.c_int32),
        ('reserved', ctypes.c_int32 * 3),
    ]


class SblGrads(ctypes.Structure):
    """Mirror of `struct SblGrads`."""
    _fields_ = [
        ('dout', ctypes.c_void_p), ('do_stride_b', ctypes.c_int64), ('do_stride_t', ctypes.c_int64),
        ('do_stride_h', ctypes.c_int64),
        ('row_stats', ctypes.c_void_p),
        ('dq', ctypes.c_void_p), ('dq_stride_b', ctypes.c_int64), ('dq_stride_t', ctypes.c_int64),
        ('dq_stride_h', ctypes.c_int64),
        ('dk', ctypes.c_void_p), ('dk_stride_b', ctypes.c_int64), ('dk_stride_s', ctypes.c_int64),
        ('dk_stride_h', ctypes.c_int64),
        ('dv', ctypes.c_void_p), ('dv_stride_b', ctypes.c_int64), ('dv_stride_s', ctypes.c_int64),
        ('dv_stride_h', ctypes.c_int64),
        ('skip', ctypes.c_int32),
        ('reserved', ctypes.c_int32 * 3),
    ]


class SblNormRotarySide(ctypes.Structure):
    """Mirror of `struct SblNormRotarySide`."""
    _fields_ = [
        ('T', ctypes.c_int32), ('H', ctypes.c_int32),
        ('x', ctypes.c_void_p), ('x_stride_b', ctypes.c_int64), ('x_stride_t', ctypes.c_int64),
        ('x_stride_h', ctypes.c_int64),
        ('y', ctypes.c_void_p), ('y_stride_b', ctypes.c_int64), ('y_stride_t', ctypes.c_int64),
        ('y_stride_h', ctypes.c_int64),
        ('dy', ctypes.c_void_p), ('dy_stride_b', ctypes.c_int64), ('dy_stride_t', ctypes.c_int64),
        ('dy_stride_h', ctypes.c_int64),
        ('weight', ctypes.c_void_p), ('dweight', ctypes.c_void_p),
        ('positions', ctypes.c_void_p), ('pos_stride_b', ctypes.c_int64), ('pos_stride_t', ctypes.c_int64),
        ('pos0', ctypes.c_int64),
    ]


class SblNormRotary(ctypes.Structure):
    """Mirror of `struct SblNormRotary`."""
    _fields_ = [
        ('dtype', ctypes.c_int32), ('weight_dtype', ctypes.c_int32),
        ('B', ctypes.c_int32), ('E', ctypes.c_int32),
        ('rotary', ctypes.c_int32), ('interleaved', ctypes.c_int32),
        ('eps', ctypes.c_double), ('theta', ctypes.c_double),
        ('side', SblNormRotarySide * 2),
        ('reserved', ctypes.c_int32 * 4),
    ]


def _packer(cls):
    """Fields in order -> an instance of the structure.  Native packing has C's alignment; for forty fields it takes a
    tenth of the time that ctypes takes to convert them one by one."""
    codes = {ctypes.c_int32: 'i', ctypes.c_int64: 'q', ctypes.c_float: 'f', ctypes.c_double: 'd', ctypes.c_void_p: 'P'}

    def fields(c):
        for _, t in c._fields_:
            if t in codes:
                yield codes[t]
            elif issubclass(t, ctypes.Array) and t._type_ in codes:
                yield codes[t._type_] * t._length_
            elif issubclass(t, ctypes.Array):
                yield from (code for _ in range(t._length_) for code in fields(t._type_))
            else:
                raise TypeError(t)

    layout = struct.Struct('@' + ''.join(fields(cls)) + '0q')
    assert layout.size == ctypes.sizeof(cls)

    def pack(*values):
        try:
            return cls.from_buffer_copy(layout.pack(*values))
        except (struct.error, OverflowError) as e:
            raise ValueError(f'sblocal_b200: a size, stride or number does not fit its field of {cls.__name__}: {e}') from e

    return pack


pack_params = _packer(SblParams)
pack_grads = _packer(SblGrads)
pack_norm_rotary = _packer(SblNormRotary)


class SblError(RuntimeError):
    """A C-ABI call returned a non-zero status."""
    def __init__(self, status, message):
        super().__init__(f'sblocal_b200 status {status}: {message}')
        self.status = status


_lock = threading.Lock()
_lib = None


def library_path():
    """In-tree library, or the file named by SBLOCAL_B200_LIB (debug builds)."""
    return os.environ.get('SBLOCAL_B200_LIB') or _build.LIB_PATH


def load():
    """Loads (once) and returns the ctypes library handle."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not os.path.exists(path):
            raise ImportError(
                f'{path} is missing: build it with `python -m fly_b200.build` (needs nvcc). '
                'sblocal_b200 has no fallback path.')
        lib = ctypes.CDLL(path)
        P = ctypes.POINTER(SblParams)
        vp, sz = ctypes.c_void_p, ctypes.c_size_t
        lib.sbl_version.restype = ctypes.c_int
        lib.sbl_version.argtypes = []
        lib.sbl_last_error.restype = ctypes.c_char_p
        lib.sbl_last_error.argtypes = []
        lib.sbl_has_tensor_path.restype = ctypes.c_int
        lib.sbl_has_tensor_path.argtypes = []
        lib.sbl_workspace_bytes.restype = ctypes.c_int
        lib.sbl_workspace_bytes.argtypes = [P, ctypes.POINTER(sz)]
        lib.sbl_forward.restype = ctypes.c_int
        lib.sbl_forward.argtypes = [P, vp, sz, vp]
        lib.sbl_key_logscale.restype = ctypes.c_int
        lib.sbl_key_logscale.argtypes = [P, vp, sz, vp, vp]
        lib.sbl_key_summary.restype = ctypes.c_int
        lib.sbl_key_summary.argtypes = [P, vp, sz, vp, vp, vp, vp]
        lib.sbl_band_forward.restype = ctypes.c_int
        lib.sbl_band_forward.argtypes = [P, vp, sz, vp, vp, vp, vp]
        lib.sbl_query_features.restype = ctypes.c_int
        lib.sbl_query_features.argtypes = [P, vp, sz, vp, vp, vp]
        lib.sbl_key_features.restype = ctypes.c_int
        lib.sbl_key_features.argtypes = [P, vp, sz, vp, vp, vp]
        lib.sbl_attention_weights.restype = ctypes.c_int
        lib.sbl_attention_weights.argtypes = [P, vp, sz, vp, vp, vp, vp]
        lib.sbl_check_status.restype = ctypes.c_int
        lib.sbl_check_status.argtypes = [P, vp, sz, vp]
        lib.sbl_status_words.restype = ctypes.c_int
        lib.sbl_status_words.argtypes = [P, ctypes.POINTER(sz)]
        lib.sbl_collect_status.restype = ctypes.c_int
        lib.sbl_collect_status.argtypes = [vp, vp, vp]
        lib.sbl_selftest_wait_timeout.restype = ctypes.c_int
        lib.sbl_selftest_wait_timeout.argtypes = [vp, sz, vp]
        lib.sbl_key_logscale_static.restype = ctypes.c_int
        lib.sbl_key_logscale_static.argtypes = [P, vp, vp]
        lib.sbl_static_last_error.restype = ctypes.c_char_p
        lib.sbl_static_last_error.argtypes = []
        G, R = ctypes.POINTER(SblGrads), ctypes.POINTER(SblNormRotary)
        lib.sbl_forward_train.restype = ctypes.c_int
        lib.sbl_forward_train.argtypes = [P, vp, sz, vp, vp]
        lib.sbl_backward_workspace_bytes.restype = ctypes.c_int
        lib.sbl_backward_workspace_bytes.argtypes = [P, ctypes.POINTER(sz)]
        lib.sbl_backward.restype = ctypes.c_int
        lib.sbl_backward.argtypes = [P, G, vp, sz, vp]
        lib.sbl_norm_rotary_forward.restype = ctypes.c_int
        lib.sbl_norm_rotary_forward.argtypes = [R, vp]
        lib.sbl_norm_rotary_workspace_bytes.restype = ctypes.c_int
        lib.sbl_norm_rotary_workspace_bytes.argtypes = [R, ctypes.POINTER(sz)]
        lib.sbl_norm_rotary_backward.restype = ctypes.c_int
        lib.sbl_norm_rotary_backward.argtypes = [R, vp, sz, vp]
        if lib.sbl_version() != ABI_VERSION:
            raise ImportError(f'{path} has ABI version {lib.sbl_version()}, expected {ABI_VERSION}: rebuild')
        _lib = lib
    return _lib


def check(status):
    """Raises the Python exception that corresponds to a C status."""
    if status == SBL_OK:
        return
    msg = load().sbl_last_error().decode('utf-8', 'replace')
    if status == SBL_ERR_INVALID_ARGUMENT:
        raise ValueError(f'sblocal_b200: {msg}')
    if status == SBL_ERR_UNSUPPORTED:
        raise NotImplementedError(f'sblocal_b200: {msg}')
    raise SblError(status, msg)
