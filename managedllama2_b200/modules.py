"""Host-side mirror of the reference's operator classes over the C ABI.

Each class keeps the name, constructor arguments and ``Forward`` argument meaning of the C# class it
stands for (src/<Name>.cs of GilesBathgate/ManagedLlama2); device buffers are torch CUDA tensors
(fp16 / int32 / uint32-as-int32) instead of ``CudaDeviceVariable``. Launch geometry is decided
inside the library, so the constructors only keep what ``Forward`` needs.
"""
import ctypes
from dataclasses import dataclass

from . import _lib


def ceil_div(a, b):
    return (a + (b - 1)) // b


def qweight_sizes(rows):
    """(weightsSize, zerosSize, scalesSize) per output row, src/QKVMatVec.cs:22-24."""
    scales = ceil_div(rows, 128)
    return ceil_div(rows, 32) * 4, ceil_div(scales, 8), scales


@dataclass
class Config:
    """src/Config.cs:6-17 (same field order as the 32-byte file header)."""
    dim: int
    hiddenDim: int
    numLayers: int
    numHeads: int
    numKVHeads: int
    vocabSize: int
    seqLength: int
    ropeTheta: float = 10000.0

    def to_struct(self):
        return _lib.ConfigStruct(self.dim, self.hiddenDim, self.numLayers, self.numHeads, self.numKVHeads,
                                 self.vocabSize, self.seqLength, self.ropeTheta)


class CudaContext:
    """Stands for ManagedCuda's ``CudaContext(deviceID)`` (src/Transformer.cs:48-49)."""

    def __init__(self, deviceID=0):
        self._lib = _lib.load()
        h = ctypes.c_void_p()
        _lib.check(self._lib.ml2_ctx_create(ctypes.c_int(deviceID), ctypes.byref(h)))
        self.handle = h
        self.device = deviceID

    def set_stream(self, stream_ptr):
        _lib.check(self._lib.ml2_ctx_set_stream(self.handle, ctypes.c_void_p(stream_ptr)))

    def set_pdl(self, enabled):
        _lib.check(self._lib.ml2_ctx_set_pdl(self.handle, ctypes.c_int(1 if enabled else 0)))

    def synchronize(self):
        _lib.check(self._lib.ml2_ctx_synchronize(self.handle))

    def set_wait_limit(self, sm_cycles):
        """Budget of every device-side wait, in SM clock cycles (default 2e10, about ten seconds)."""
        _lib.check(self._lib.ml2_ctx_set_wait_limit(self.handle, ctypes.c_longlong(int(sm_cycles))))

    def status(self):
        err, det = ctypes.c_uint(), ctypes.c_uint()
        _lib.check(self._lib.ml2_ctx_status(self.handle, ctypes.byref(err), ctypes.byref(det)))
        return err.value, det.value

    @property
    def launch_count(self):
        return int(self._lib.ml2_ctx_launch_count(self.handle))

    def close(self):
        if self.handle:
            self._lib.ml2_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _ptr(t, offset_elems=0):
    """Device pointer of a torch tensor, optionally offset by elements (OffsetPointer, src/Extensions.cs:20-21)."""
    return ctypes.c_void_p(t.data_ptr() + offset_elems * t.element_size())


class QWeight:
    """src/QWeight.cs:5-10: Weight (uint32), Zeros (uint32), Scales (fp16) device arrays."""

    def __init__(self, Weight, Zeros, Scales):
        self.Weight, self.Zeros, self.Scales = Weight, Zeros, Scales

    def struct(self):
        return _lib.QWeightStruct(self.Weight.data_ptr(), self.Zeros.data_ptr(), self.Scales.data_ptr())


class Module:
    """src/Module.cs:7-26. The PTX-per-module loading is replaced by the shared library."""

    def __init__(self, cudaContext):
        self.ctx = cudaContext
        self.lib = cudaContext._lib

    @staticmethod
    def CeilDiv(a, b):
        return ceil_div(a, b)


class MatVec(Module):
    """src/MatVec.cs:6-17."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, output, input, matrix, rows, cols):
        _lib.check(self.lib.ml2_matvec_f16(self.ctx.handle, _ptr(output), _ptr(input), _ptr(matrix), rows, cols))


class QKVMatVec(Module):
    """src/QKVMatVec.cs:7-32."""

    def __init__(self, cudaContext, config):
        super().__init__(cudaContext)
        self.kvDim = config.dim * config.numKVHeads // config.numHeads

    def Forward(self, queryOutput, keyOutput, valueOutput, input, query, key, value, rows, cols, layerOffset, pos):
        offset = layerOffset + pos * self.kvDim  # :25
        q, k, v = query.struct(), key.struct(), value.struct()
        _lib.check(self.lib.ml2_qkv_matvec_int4(self.ctx.handle, _ptr(queryOutput), _ptr(keyOutput, offset),
                                                _ptr(valueOutput, offset), _ptr(input), ctypes.byref(q),
                                                ctypes.byref(k), ctypes.byref(v), rows, cols))


class MatVecSwiGLU(Module):
    """src/MatVecSwiGLU.cs:6-24."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, output, input, g, u, rows, cols):
        gs, us = g.struct(), u.struct()
        _lib.check(self.lib.ml2_matvec_swiglu_int4(self.ctx.handle, _ptr(output), _ptr(input), ctypes.byref(gs),
                                                   ctypes.byref(us), rows, cols))


class MatVecResidual(Module):
    """src/MatVecResidual.cs:6-24."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, output, input, matrix, rows, cols):
        m = matrix.struct()
        _lib.check(self.lib.ml2_matvec_residual_int4(self.ctx.handle, _ptr(output), _ptr(input), ctypes.byref(m), rows,
                                                     cols))


class MatVecStrided(Module):
    """src/MatVecStrided.cs:7-19. ``seqLength`` is the live length (pos + 1)."""

    def __init__(self, cudaContext, config):
        super().__init__(cudaContext)
        self.numHeads = config.numHeads

    def Forward(self, attention, query, key, headSize, dim, seqLength, layerOffset, scale):
        _lib.check(self.lib.ml2_matvec_strided(self.ctx.handle, _ptr(attention), _ptr(query), _ptr(key, layerOffset),
                                               headSize, dim, self.numHeads, seqLength, ctypes.c_float(scale)))


class VecMat(Module):
    """src/VecMat.cs:7-19."""

    def __init__(self, cudaContext, config):
        super().__init__(cudaContext)
        self.numHeads = config.numHeads

    def Forward(self, output, value, attention, headSize, dim, seqLength, layerOffset):
        _lib.check(self.lib.ml2_vecmat(self.ctx.handle, _ptr(output), _ptr(value, layerOffset), _ptr(attention),
                                       headSize, dim, self.numHeads, seqLength))


class RMSNorm(Module):
    """src/RMSNorm.cs:5-15."""

    def Forward(self, output, input, weights, size, eps=1e-5):
        _lib.check(self.lib.ml2_rmsnorm(self.ctx.handle, _ptr(output), _ptr(input), _ptr(weights), size,
                                        ctypes.c_float(eps)))


class RoPERotation(Module):
    """src/RoPERotation.cs:6-24."""

    def __init__(self, cudaContext, config):
        super().__init__(cudaContext)
        self.kvDim = config.dim * config.numKVHeads // config.numHeads
        self.numHeads = config.numHeads

    def Forward(self, query, key, numKVHeads, headSize, pos, layerOffset, theta):
        offset = layerOffset + pos * self.kvDim  # :22
        _lib.check(self.lib.ml2_rope(self.ctx.handle, _ptr(query), _ptr(key, offset), self.numHeads, numKVHeads,
                                     headSize, pos, ctypes.c_float(theta)))


class Softmax(Module):
    """src/Softmax.cs:5-15."""

    def __init__(self, cudaContext, config):
        super().__init__(cudaContext)
        self.numHeads = config.numHeads

    def Forward(self, attention, seqLength):
        _lib.check(self.lib.ml2_softmax(self.ctx.handle, _ptr(attention), self.numHeads, seqLength))


class Embedding(Module):
    """src/Embedding.cs:5-15."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, output, table, size, tokens, pos):
        _lib.check(self.lib.ml2_embedding(self.ctx.handle, _ptr(output), _ptr(table), size, _ptr(tokens), pos))


class Argmax(Module):
    """src/Argmax.cs:5-15."""

    def Forward(self, logits, vocabSize, tokens, nextPos, generateToken):
        _lib.check(self.lib.ml2_argmax(self.ctx.handle, _ptr(logits), vocabSize, _ptr(tokens), nextPos,
                                       1 if generateToken else 0))


class SoftmaxLogits(Module):
    """src/SoftmaxLogits.cs:5-16."""

    def Forward(self, logits, size, temperature, indices):
        _lib.check(self.lib.ml2_softmax_logits(self.ctx.handle, _ptr(logits), size, ctypes.c_float(temperature), _ptr(indices)))


class Sort(Module):
    """src/Sort.cs:5-16 (descending by key, values carried; any size up to 32768)."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, logits, indices, size):
        _lib.check(self.lib.ml2_sort(self.ctx.handle, _ptr(logits), _ptr(indices), size))


class CumulativeSum(Module):
    """src/CumulativeSum.cs:5-16."""

    def __init__(self, cudaContext, config=None):
        super().__init__(cudaContext)

    def Forward(self, logits, size):
        _lib.check(self.lib.ml2_cumulative_sum(self.ctx.handle, _ptr(logits), size))


class SampleTopP(Module):
    """src/SampleTopP.cs:5-16."""

    def Forward(self, logits, indices, size, threshold, tokens, nextPos):
        _lib.check(self.lib.ml2_sample_top_p(self.ctx.handle, _ptr(logits), _ptr(indices), size, ctypes.c_float(threshold),
                                             _ptr(tokens), nextPos))


# ---- batched decoding over a paged cache: no counterpart in the reference, which decodes one sequence ------------------------

_torch = None  # fetched by the first operator that is made: importing this package does not import torch


def _use_torch():
    global _torch
    if _torch is None:
        import torch
        _torch = torch


def _dtype_code(t, what):
    if t.dtype is _torch.float16:
        return 0  # ML2_F16
    if t.dtype is _torch.bfloat16:
        return 1  # ML2_BF16
    raise ValueError("%s: type %s is neither float16 nor bfloat16" % (what, t.dtype))


def _rows(ctx, what, t, width, dtype):
    """Checks a [rows][width] tensor whose rows may be apart (a slice of columns); returns its rows and their stride in elements."""
    if t.dtype is not dtype or t.get_device() != ctx.device:
        raise ValueError("%s: expected %s on cuda:%d, got %s on %s" % (what, dtype, ctx.device, t.dtype, t.device))
    if t.dim() == 2:
        rows, columns = t.shape
        stride, step = t.stride()
        if columns == width and (step == 1 or width == 1):
            return rows, stride if rows > 1 else max(width, stride)
    raise ValueError("%s: expected [rows][%d] with neighbouring columns, got %s with strides %s" % (what, width, tuple(t.shape), t.stride()))


def _ints(ctx, what, t, count):
    """Checks a contiguous int32 tensor of at least `count` entries; returns its device pointer."""
    if t.dtype is not _torch.int32 or t.get_device() != ctx.device or not t.is_contiguous() or t.numel() < count:
        raise ValueError("%s: expected a contiguous int32 tensor of at least %d entries on cuda:%d, got %s %s on %s"
                         % (what, count, ctx.device, tuple(t.shape), t.dtype, t.device))
    return t.data_ptr()


class BlockTables(Module):
    """Block tables and slot maps of a batch from its request lengths (``ml2_block_tables``). All arrays are int32.

    ``table`` is [requests][pages of the longest request], ``freePages`` the stack of free pages with room for every page of
    the cache, ``slots`` and ``positions`` have one entry for every row of the step's token buffer."""

    def __init__(self, cudaContext, pageSize):
        super().__init__(cudaContext)
        _use_torch()
        self.pageSize = pageSize
        self._call = _lib.BLOCK_TABLES.entry(self.lib.ml2_block_tables)

    def Forward(self, lengths, newLengths, table, freePages, freeCount, lengthsOut, freeCountOut, queryStart, slots, positions, refused,
                positionOffset=0):
        c, n, rows = self.ctx, newLengths.numel(), slots.numel()
        if table.dim() != 2 or table.shape[0] != n:
            raise ValueError("table: expected [%d][pages], got %s" % (n, tuple(table.shape)))
        rc = self._call(c.handle, _lib.BLOCK_TABLES.pack(
            _ints(c, "lengths", lengths, n), _ints(c, "newLengths", newLengths, n), _ints(c, "table", table, 1),
            _ints(c, "freePages", freePages, 1), _ints(c, "freeCount", freeCount, 1), _ints(c, "lengthsOut", lengthsOut, n),
            _ints(c, "freeCountOut", freeCountOut, 1), _ints(c, "queryStart", queryStart, n + 1), _ints(c, "slots", slots, rows),
            _ints(c, "positions", positions, rows), _ints(c, "refused", refused, n), n, self.pageSize, table.shape[1], freePages.numel(), rows,
            positionOffset))
        if rc:
            _lib.check(rc)


class QKNormRoPE(Module):
    """Norm of query and key heads, rotation and cache write of a batch of tokens (``ml2_qk_norm_rope``).

    ``query``, ``key`` and ``value`` are [tokens][heads * headSize] and may be columns of one tensor; the caches are
    [rows][numKVHeads * headSize]. ``queryWeight`` and ``keyWeight`` are None for models without head norms. ``queryOutput`` may be
    ``query`` (with its strides). Heads of any multiple of 16 up to 256; ``PrefixAttention`` reads those of 64 and 128."""

    def __init__(self, cudaContext, config, rotarySize=None):
        super().__init__(cudaContext)
        _use_torch()
        self.numHeads, self.numKVHeads, self.theta = config.numHeads, config.numKVHeads, config.ropeTheta
        self.headSize = config.dim // config.numHeads
        self.rotarySize = self.headSize if rotarySize is None else rotarySize
        self._call = _lib.QK_NORM_ROPE.entry(self.lib.ml2_qk_norm_rope)

    def _weight(self, what, w, dtype):
        if w is None:
            return 0
        if w.dtype is not dtype or w.get_device() != self.ctx.device or not w.is_contiguous() or w.numel() != self.headSize:
            raise ValueError("%s: expected %d contiguous %s on cuda:%d" % (what, self.headSize, dtype, self.ctx.device))
        return w.data_ptr()

    def Forward(self, queryOutput, keyCache, valueCache, query, key, value, queryWeight, keyWeight, positions, slots, eps=1e-5):
        c, dtype = self.ctx, query.dtype
        code, width, kvWidth = _dtype_code(query, "query"), self.numHeads * self.headSize, self.numKVHeads * self.headSize
        n, queryStride = _rows(c, "query", query, width, dtype)
        nk, keyStride = _rows(c, "key", key, kvWidth, dtype)
        nv, valueStride = _rows(c, "value", value, kvWidth, dtype)
        no, outStride = _rows(c, "queryOutput", queryOutput, width, dtype)
        cache = _rows(c, "keyCache", keyCache, kvWidth, dtype)
        if _rows(c, "valueCache", valueCache, kvWidth, dtype) != cache:
            raise ValueError("keyCache and valueCache must have the same rows and strides")
        if nk != n or nv != n or no < n:
            raise ValueError("query, key, value and queryOutput must have the same rows")
        rc = self._call(c.handle, _lib.QK_NORM_ROPE.pack(
            queryOutput.data_ptr(), keyCache.data_ptr(), valueCache.data_ptr(), query.data_ptr(), key.data_ptr(), value.data_ptr(),
            self._weight("queryWeight", queryWeight, dtype), self._weight("keyWeight", keyWeight, dtype), _ints(c, "positions", positions, n),
            _ints(c, "slots", slots, n), outStride, cache[1], cache[0], queryStride, keyStride, valueStride, code, n, self.numHeads,
            self.numKVHeads, self.headSize, self.rotarySize, self.theta, eps))
        if rc:
            _lib.check(rc)


class PrefixAttention(Module):
    """Attention of a batch that shares a prefix (``ml2_prefix_attention``).

    ``prefixKey`` and ``prefixValue`` are the shared rows, [length][numKVHeads * headSize] (a slice of a ``Transformer``'s own
    caches will do; None: nothing is shared), ``keyCache`` and ``valueCache`` the pages of all requests. Runs on the stream that the
    context was given, behind what a ``Transformer`` of the context has queued. Heads of 64 or 128; the config's ``dim`` is
    taken as numHeads heads of one size, so a model whose heads have another one gets a config of its own here."""

    def __init__(self, cudaContext, config, pageSize):
        super().__init__(cudaContext)
        _use_torch()
        self.numHeads, self.numKVHeads, self.pageSize = config.numHeads, config.numKVHeads, pageSize
        self.headSize = config.dim // config.numHeads
        self._sizes = {}
        self._call = _lib.PREFIX_ATTENTION.entry(self.lib.ml2_prefix_attention)

    def WorkspaceBytes(self, rows, requests, prefixLength, maxLength):
        """Size of the workspace for a call of these sizes; calls that may overlap need one each."""
        sizes = (rows, requests, prefixLength, maxLength)
        if sizes not in self._sizes:
            n = ctypes.c_size_t()
            _lib.check(self.lib.ml2_prefix_attention_workspace(ctypes.c_void_p(getattr(self.ctx.handle, "value", self.ctx.handle)), *sizes,
                                                               self.numHeads, self.numKVHeads, self.headSize, ctypes.byref(n)))
            if len(self._sizes) > 1000:
                self._sizes.clear()
            self._sizes[sizes] = n.value
        return self._sizes[sizes]

    def Forward(self, output, query, prefixKey, prefixValue, keyCache, valueCache, table, lengths, queryStart, workspace, maxLength,
                lse=None, scale=None):
        c, dtype, n = self.ctx, query.dtype, lengths.numel()
        code, width, kvWidth = _dtype_code(query, "query"), self.numHeads * self.headSize, self.numKVHeads * self.headSize
        rows, queryStride = _rows(c, "query", query, width, dtype)
        outRows, outStride = _rows(c, "output", output, width, dtype)
        cache = _rows(c, "keyCache", keyCache, kvWidth, dtype)
        if _rows(c, "valueCache", valueCache, kvWidth, dtype) != cache:
            raise ValueError("keyCache and valueCache must have the same rows and strides")
        if outRows < rows or table.dim() != 2 or table.shape[0] != n:
            raise ValueError("output needs %d rows and table %d; got %d and %s" % (rows, n, outRows, tuple(table.shape)))
        prefix, prefixKeyPtr, prefixValuePtr = (0, kvWidth), 0, 0
        if (prefixKey is not None and prefixKey.numel()) or (prefixValue is not None and prefixValue.numel()):
            if prefixKey is None or prefixValue is None:
                raise ValueError("prefixKey and prefixValue come together or not at all")
            prefix = _rows(c, "prefixKey", prefixKey, kvWidth, dtype)
            if _rows(c, "prefixValue", prefixValue, kvWidth, dtype) != prefix:
                raise ValueError("prefixKey and prefixValue must have the same rows and strides")
            prefixKeyPtr, prefixValuePtr = prefixKey.data_ptr(), prefixValue.data_ptr()
        lsePtr = 0
        if lse is not None:
            if lse.dtype is not _torch.float32 or lse.get_device() != c.device or not lse.is_contiguous() or lse.numel() < rows * self.numHeads:
                raise ValueError("lse: expected contiguous float32 [%d][%d] on cuda:%d" % (rows, self.numHeads, c.device))
            lsePtr = lse.data_ptr()
        if workspace.get_device() != c.device or not workspace.is_contiguous():
            raise ValueError("workspace: expected a contiguous tensor on cuda:%d" % c.device)
        rc = self._call(c.handle, _lib.PREFIX_ATTENTION.pack(
            output.data_ptr(), lsePtr, query.data_ptr(), prefixKeyPtr, prefixValuePtr, keyCache.data_ptr(), valueCache.data_ptr(),
            _ints(c, "table", table, 1), _ints(c, "lengths", lengths, n), _ints(c, "queryStart", queryStart, n + 1), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), outStride, queryStride, prefix[1], cache[1], cache[0], code, rows, n, prefix[0],
            maxLength, self.pageSize, table.shape[1], self.numHeads, self.numKVHeads, self.headSize,
            self.headSize ** -0.5 if scale is None else scale))
        if rc:
            _lib.check(rc)
