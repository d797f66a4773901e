"""ctypes loader for libml2b200.so. There is no fallback: a missing library or symbol raises."""
import ctypes
import os
import re
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libml2b200.so")
HEADER_PATH = os.path.join(os.path.dirname(HERE), "include", "ml2b200.h")

_lib = None


class Ml2Error(RuntimeError):
    def __init__(self, code, text):
        super().__init__("ml2b200 error %d: %s" % (code, text))
        self.code = code


def declared_symbols():
    """Names of every function include/ml2b200.h declares."""
    text = open(HEADER_PATH).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(ml2_[a-z0-9_]+)\s*\(", text)))


def load():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError("%s is missing: build it with `python -m managedllama2_b200.build` "
                              "(there is no CPU or PyTorch fallback)" % LIB_PATH)
        lib = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_GLOBAL)
        lib.ml2_last_error.restype = ctypes.c_char_p
        lib.ml2_ctx_launch_count.restype = ctypes.c_longlong
        _lib = lib
    return _lib


def check(rc):
    if rc != 0:
        raise Ml2Error(rc, load().ml2_last_error().decode("utf-8", "replace"))


class QWeightStruct(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("zeros", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


class ConfigStruct(ctypes.Structure):
    _fields_ = [("dim", ctypes.c_int32), ("hidden_dim", ctypes.c_int32), ("n_layers", ctypes.c_int32),
                ("n_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32), ("vocab_size", ctypes.c_int32),
                ("seq_len", ctypes.c_int32), ("rope_theta", ctypes.c_float)]


class Arguments:
    """The argument struct of a C entry: its members and their kinds (p pointer, l long long / size_t, i int, f float), packed
    as the C compiler lays them out. Bytes from ``struct`` cost a third of a call with as many ctypes arguments."""

    def __init__(self, *members):
        self.names, self.kinds = [], ""
        for kind, names in members:
            names = names.split()
            self.names += names
            self.kinds += kind * len(names)
        # 0P: the end is padded to a pointer's alignment, as the struct's is
        self._pack = struct.Struct("@" + self.kinds.replace("p", "P").replace("l", "q") + "0P").pack

    def pack(self, *values):
        try:
            return self._pack(*values)
        except struct.error as e:
            wrong = [n for n, k, v in zip(self.names, self.kinds, values) if k == "i" and isinstance(v, int) and not -2**31 <= v < 2**31]
            raise ValueError("%s: passes 32 bits" % ", ".join(wrong) if wrong else str(e)) from None

    def entry(self, function):
        function.argtypes = [ctypes.c_void_p, ctypes.c_char_p]
        function.restype = ctypes.c_int
        return function


BLOCK_TABLES = Arguments(
    ("p", "lengths new_lengths table free_pages free_count lengths_out free_count_out query_start slots positions refused"),
    ("i", "n_requests page_size table_stride n_pages max_tokens position_offset"))
QK_NORM_ROPE = Arguments(
    ("p", "query_out key_cache value_cache query key value query_weight key_weight positions slots"),
    ("l", "query_out_stride cache_stride cache_rows query_stride key_stride value_stride"),
    ("i", "dtype n_tokens n_heads n_kv_heads head_size rotary_size"), ("f", "theta eps"))
PREFIX_ATTENTION = Arguments(
    ("p", "out lse query prefix_key prefix_value key_cache value_cache table lengths query_start workspace"),
    ("l", "workspace_bytes out_stride query_stride prefix_stride cache_stride cache_rows"),
    ("i", "dtype n_rows n_requests prefix_length max_length page_size table_stride n_heads n_kv_heads head_size"), ("f", "scale"))
