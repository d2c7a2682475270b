"""ctypes bindings of ``build/libqvelox.so`` (sm_100a build of the hot path).

``load_library`` binds the same symbols with the same ctypes signatures as the
reference loader (cristianku/redshift ``qvelox/runtime.py:6-22``), then the
additive entry points of ``include/runtime.h``.  A missing library raises at
once: there is no CPU fallback anywhere in this package.

``HotPath`` is a thin convenience layer over the device-resident entry points
for callers that hold their buffers as torch CUDA tensors (torch supplies the
device memory and the current stream; all arithmetic runs in the library's
own kernels).
"""
import ctypes as ct
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
DEFAULT_LIBRARY = ROOT / 'build' / 'libqvelox.so'

_P, _I, _F, _S = ct.c_void_p, ct.c_int, ct.c_float, ct.c_size_t

# The reference loader's table (qvelox/runtime.py:11-17), unchanged.
REFERENCE_SIGNATURES = {
    'qv_test_mm': [_P] * 3 + [_I] * 4,
    'qv_test_mm_fast': [_P] * 3 + [_I] * 4,
    'qv_test_norm': [_P] * 3 + [_I] * 2 + [_F],
    'qv_test_delta': [_P] * 11 + [_I] * 4 + [_F],
    'qv_test_attention': [_P] * 8 + [_I] * 2 + [_F],
}
# Model ABI of the reference (qvelox/runtime.py:37-46).
MODEL_SIGNATURES = {
    'qv_create': [ct.POINTER(_P), ct.c_char_p, _I, _F],
    'qv_upload': [_P, _I, ct.c_uint64, ct.c_uint64],
    'qv_evaluate': [_P, ct.POINTER(_I), _I, ct.POINTER(_F)],
    'qv_verify': [_P, ct.POINTER(_I), _I, ct.POINTER(_F)],
    'qv_commit': [_P, _I],
    'qv_advance': [_P, ct.POINTER(_I), _I, ct.POINTER(_I)],
    'qv_position': [_P, ct.POINTER(_I)],
    'qv_reset': [_P], 'qv_checkpoint': [_P], 'qv_restore': [_P],
}
# Additive entry points (include/runtime.h, part 2).
ADDITIVE_SIGNATURES = {
    'qv_test_attention_prefill': ([_P] * 8 + [_I] * 2 + [_F], _I),
    'qv_test_delta_prefill': ([_P] * 11 + [_I] * 4 + [_F], _I),
    'qv_attention_workspace': ([_I, _I], _S),
    'qv_attention': ([_P] * 8 + [_I, _I, _F, _P, _S, _P], _I),
    'qv_delta': ([_P] * 11 + [_I] * 4 + [_F, _P], _I),
    'qv_delta_trace_floats': ([_I, _I, _I], _S),
    'qv_mm_weight_bytes': ([_I, _I, _I], _S),
    'qv_copy_spans': ([_P, _P, _P, _I, _P], _I),
    'qv_mm': ([_P] * 3 + [_I] * 5 + [_P], _I),
    'qv_delta_verify': ([_P] * 11 + [_I] * 4 + [_F] + [_P] * 4, _I),
    'qv_delta_commit': ([_P] * 5 + [_I] * 5 + [_P], _I),
    'qv_attention_shard_workspace': ([_I, _I], _S),
    'qv_attention_shard': ([_P] * 4 + [_I, _I] + [_P] * 5 + [_I, _I, _F, _P, _S, _P], _I),
    'qv_attention_merge': ([_P] * 3 + [_I, _I, _P, _P], _I),
    'qv_attention_exchange_bytes': ([_I], _S),
    'qv_attention_shard_exchange': ([_P] * 3 + [_I, _I] + [_P] * 5 + [_I, _I, _F] + [_P, _I, _I, _I, _P, _S, _P], _I),
    'qv_prefill_attention': ([_P] * 5 + [_I, _I, _P], _I),
    'qv_delta_core': ([_P] * 9 + [_I] * 4 + [_P], _I),
    'qv_delta_chunked_workspace': ([_I, _I], _S),
    'qv_delta_chunked': ([_P] * 9 + [_I] * 4 + [_P, _S, _P], _I),
    'qv_delta_prefill_workspace': ([_I, _I, _I], _S),
    'qv_delta_prefill': ([_P] * 11 + [_I] * 4 + [_F, _P, _S, _P], _I),
    'qv_status': ([], _I),
    'qv_norm8': ([_P] * 7 + [_I, _I, _F, _P], _I),
    'qv_quantize8': ([_P] * 3 + [_I, _I, _P], _I),
    'qv_mm8': ([_P] * 5 + [_I] * 3 + [_P], _I),
    'qv_attention8_workspace': ([_I, _I], _S),
    'qv_attention8': ([_P] * 5 + [_I, _P, _P, _I] + [_P] * 5 + [_I, _I, _F, _P, _S, _P], _I),
    'qv_cache8_pack': ([_P] * 6 + [_I] * 3 + [_P], _I),
    'qv_cache8_unpack': ([_P] * 6 + [_I] * 2 + [_P], _I),
    'qv_attention_noalloc': ([_P] * 8 + [_I, _I, _F, _P], _I),
}


def load_library(path=None):
    """Load the library and declare every exported signature.

    Raises ``OSError`` when the library is missing: build it with
    ``python -m redshift_b200.build``.
    """
    path = Path(path) if path is not None else DEFAULT_LIBRARY
    if not path.exists():
        raise OSError(f'{path} is missing; build it with `python -m redshift_b200.build`')
    lib = ct.CDLL(str(path.resolve()))
    lib.qv_error.argtypes = []
    lib.qv_error.restype = ct.c_char_p
    for table in (REFERENCE_SIGNATURES, MODEL_SIGNATURES):
        for name, signature in table.items():
            fn = getattr(lib, name)
            fn.argtypes = signature
            fn.restype = _I
    lib.qv_destroy.argtypes = [_P]
    lib.qv_destroy.restype = None
    for name, (signature, restype) in ADDITIVE_SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = signature
        fn.restype = restype
    return lib


class NativeError(RuntimeError):
    """A library call returned -1; the message is ``qv_error()``."""


# Host-side checks of the 8-bit calls, which take their sizes from the tensors: a wrong shape, element
# size, layout or device is refused here, before an address reaches a kernel.  They run on every call of
# a decode step, so they ask a tensor only what is cheap to ask (a CPU tensor's device number is -1).
class ElementTypes:
    """The element types that the 8-bit calls take; e4m3 codes and workspaces may also be plain bytes."""

    def __init__(self):
        import torch
        self.float = (torch.float32,)
        self.half = (torch.float16,)
        self.int8 = (torch.int8,)
        self.e4m3 = (torch.float8_e4m3fn, torch.uint8)
        self.bytes = (torch.uint8, torch.int8)


def need_tensor(t, types, shape, name, device):
    if t.dtype not in types or t.shape != shape or t.get_device() != device or device < 0 or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous CUDA tensor of shape {list(shape)} and type '
                         + ' or '.join(str(x) for x in types) + (f' on device {device}' if device >= 0 else ''))


def need_cache8(types, key_codes, key_scales, value_codes, value_scales, end, device):
    blocks = key_codes.shape[0]
    need_tensor(key_codes, types.int8, (blocks, 4, 64, 256), 'key_codes', device)
    need_tensor(value_codes, types.int8, (blocks, 4, 64, 256), 'value_codes', device)
    need_tensor(key_scales, types.float, (blocks, 4), 'key_scales', device)
    need_tensor(value_scales, types.float, (blocks, 4), 'value_scales', device)
    if end > 64 * blocks:
        raise ValueError(f'the cache holds {blocks} blocks of 64 rows, not {end} rows')


class HotPath:
    """Device-resident hot-path calls on torch CUDA tensors.

    Every method validates shapes/dtypes on the host, then calls one entry
    point of the library on torch's current CUDA stream.  Buffers are used in
    place; nothing is copied or converted here.
    """

    def __init__(self, library=None):
        self.lib = load_library(library)
        self._workspace = None
        self._workspaces8 = {}
        self._types = ElementTypes()

    # -- helpers ---------------------------------------------------------
    def check(self, code):
        if code:
            raise NativeError(self.lib.qv_error().decode('utf-8', errors='replace'))

    @staticmethod
    def _stream():
        import torch
        return ct.c_void_p(torch.cuda.current_stream().cuda_stream)

    @staticmethod
    def capturing(device=None):
        """Whether torch's current stream of `device` (of the current device) is being captured into a graph."""
        import torch
        if device is None or getattr(device, 'index', device) == torch._C._cuda_getDevice():
            return torch.cuda.is_current_stream_capturing()
        with torch.cuda.device(device):
            return torch.cuda.is_current_stream_capturing()

    @staticmethod
    def _ptr(t):
        return ct.c_void_p(t.data_ptr()) if t is not None else None

    def workspace(self, nbytes, device):
        """A cached device workspace of at least ``nbytes`` bytes, zero-filled when it is made (the
        attention workspace's barrier words must start at zero; the calls keep them so)."""
        import torch
        if self._workspace is None or self._workspace.numel() < nbytes or self._workspace.device != device:
            self._workspace = torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)
        return self._workspace

    # -- attention --------------------------------------------------------
    def attention(self, out, key_cache, value_cache, q_gate, key, value, q_norm, k_norm,
                  batch, position, epsilon=1e-6, workspace=None):
        """One attention layer (prepare + decode/verify or prefill) in place."""
        need = self.lib.qv_attention_workspace(batch, position)
        ws = workspace if workspace is not None else self.workspace(need, out.device)
        p = self._ptr
        self.check(self.lib.qv_attention(p(out), p(key_cache), p(value_cache), p(q_gate), p(key), p(value),
                                         p(q_norm), p(k_norm), batch, position, epsilon, p(ws),
                                         ws.numel() * ws.element_size(), self._stream()))

    def attention_shard(self, partial, lse, key_cache, value_cache, shard_begin, shard_rows, q_gate, key,
                        value, q_norm, k_norm, batch, position, epsilon=1e-6, workspace=None):
        need = self.lib.qv_attention_shard_workspace(batch, shard_rows)
        ws = workspace if workspace is not None else self.workspace(need, partial.device)
        p = self._ptr
        self.check(self.lib.qv_attention_shard(p(partial), p(lse), p(key_cache), p(value_cache), shard_begin,
                                               shard_rows, p(q_gate), p(key), p(value), p(q_norm), p(k_norm),
                                               batch, position, epsilon, p(ws), ws.numel() * ws.element_size(),
                                               self._stream()))

    def attention_shard_exchange(self, out, key_cache, value_cache, shard_begin, shard_rows, q_gate, key, value,
                                 q_norm, k_norm, batch, position, peers, world, rank, sequence, epsilon=1e-6,
                                 workspace=None):
        """Shard attention + peer-memory exchange + merge (``peers``: int64 device tensor of buffer
        addresses; ``sequence``: the call's number on these buffers, +1 per call, the same on every rank)."""
        need = self.lib.qv_attention_shard_workspace(batch, shard_rows)
        ws = workspace if workspace is not None else self.workspace(need, out.device)
        p = self._ptr
        self.check(self.lib.qv_attention_shard_exchange(
            p(out), p(key_cache), p(value_cache), shard_begin, shard_rows, p(q_gate), p(key), p(value), p(q_norm),
            p(k_norm), batch, position, epsilon, p(peers), world, rank, sequence, p(ws), ws.numel() * ws.element_size(),
            self._stream()))

    def attention_merge(self, out, partials, lses, shards, batch, q_gate):
        p = self._ptr
        self.check(self.lib.qv_attention_merge(p(out), p(partials), p(lses), shards, batch, p(q_gate),
                                               self._stream()))

    def prefill_attention(self, out, q, key_cache, value_cache, tokens, position=0, lse=None):
        p = self._ptr
        self.check(self.lib.qv_prefill_attention(p(out), p(lse), p(q), p(key_cache), p(value_cache), tokens,
                                                 position, self._stream()))

    # -- DeltaNet ---------------------------------------------------------
    def delta(self, out, state, history, qkv, gate, alpha, beta, conv, decay, bias, norm,
              batch, key_heads, value_heads, dim, epsilon=1e-6):
        p = self._ptr
        self.check(self.lib.qv_delta(p(out), p(state), p(history), p(qkv), p(gate), p(alpha), p(beta),
                                     p(conv), p(decay), p(bias), p(norm), batch, key_heads, value_heads, dim,
                                     epsilon, self._stream()))

    def copy_spans(self, pairs):
        """qv_copy_spans over [(dst_tensor, src_tensor[, bytes]), ...] (whole tensors by default)."""
        import ctypes
        n = len(pairs)
        dst = (ctypes.c_void_p * n)(*[d.data_ptr() for d, s, *_ in pairs])
        src = (ctypes.c_void_p * n)(*[s.data_ptr() for d, s, *_ in pairs])
        nb = (ctypes.c_size_t * n)(*[(rest[0] if rest else s.numel() * s.element_size()) for d, s, *rest in pairs])
        self.check(self.lib.qv_copy_spans(dst, src, nb, n, self._stream()))

    def mm(self, out, weights, x, kind, batch, width, rows, fast=False):
        """qv_mm: out [batch][rows] = W x for a block-quantized W on the device."""
        p = self._ptr
        self.check(self.lib.qv_mm(p(out), p(weights), p(x), kind, batch, width, rows, int(bool(fast)),
                                  self._stream()))

    def delta_verify(self, out, state, history, qkv, gate, alpha, beta, conv, decay, bias, norm,
                     batch, key_heads, value_heads, dim, saved_state, saved_history, trace, epsilon=1e-6):
        """qv_delta_verify: qv_delta that also saves the start state / history and
        writes the transition trace that qv_delta_commit replays."""
        p = self._ptr
        self.check(self.lib.qv_delta_verify(p(out), p(state), p(history), p(qkv), p(gate), p(alpha), p(beta),
                                            p(conv), p(decay), p(bias), p(norm), batch, key_heads, value_heads,
                                            dim, epsilon, p(saved_state), p(saved_history), p(trace),
                                            self._stream()))

    def delta_commit(self, state, history, saved_state, saved_history, trace, accepted, batch,
                     key_heads, value_heads, dim):
        """qv_delta_commit: keep the first `accepted` tokens of a recorded verify."""
        p = self._ptr
        self.check(self.lib.qv_delta_commit(p(state), p(history), p(saved_state), p(saved_history), p(trace),
                                            accepted, batch, key_heads, value_heads, dim, self._stream()))

    def delta_core(self, out, state, q, k, v, alpha, beta, decay, bias, tokens, key_heads, value_heads, dim):
        p = self._ptr
        self.check(self.lib.qv_delta_core(p(out), p(state), p(q), p(k), p(v), p(alpha), p(beta), p(decay),
                                          p(bias), tokens, key_heads, value_heads, dim, self._stream()))

    def delta_chunked(self, out, state, q, k, v, alpha, beta, decay, bias, tokens, key_heads, value_heads, dim,
                      workspace=None):
        """qv_delta_chunked; allocates the workspace when none is given."""
        p = self._ptr
        need = self.lib.qv_delta_chunked_workspace(tokens, value_heads)
        if workspace is None:
            import torch
            workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=out.device)
        self.check(self.lib.qv_delta_chunked(p(out), p(state), p(q), p(k), p(v), p(alpha), p(beta), p(decay),
                                             p(bias), tokens, key_heads, value_heads, dim, p(workspace),
                                             workspace.numel() * workspace.element_size(), self._stream()))

    def delta_prefill(self, out, state, history, qkv, gate, alpha, beta, conv, decay, bias, norm,
                      tokens, key_heads, value_heads, dim, epsilon=1e-6, workspace=None):
        """qv_delta_prefill: the DeltaNet layer over a long block in the chunked form; allocates the
        workspace when none is given."""
        p = self._ptr
        need = self.lib.qv_delta_prefill_workspace(tokens, key_heads, value_heads)
        if workspace is None:
            import torch
            workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=out.device)
        self.check(self.lib.qv_delta_prefill(p(out), p(state), p(history), p(qkv), p(gate), p(alpha), p(beta),
                                             p(conv), p(decay), p(bias), p(norm), tokens, key_heads, value_heads,
                                             dim, epsilon, p(workspace), workspace.numel() * workspace.element_size(),
                                             self._stream()))

    # -- 8-bit serving ------------------------------------------------------
    def _call(self, device, function, *args):
        """function(*args, stream) with device number `device` current, on torch's current stream of it."""
        import torch
        stream = torch._C._cuda_getCurrentRawStream(device)      # what torch.cuda.current_stream(device) wraps
        if torch._C._cuda_getDevice() == device:
            code = function(*args, stream)
        else:
            with torch.cuda.device(device):
                code = function(*args, stream)
        if code:
            self.check(code)

    def norm8(self, codes, scales, x, weights, residual=None, residual_out=None, normed=None, epsilon=1e-6):
        """qv_norm8: e4m3 codes [tokens][width] and scales [ceil(width/128)][tokens] of the RMSNorm of
        x (+ residual); residual_out and normed, where given, receive the sum and the norm in fp32."""
        types = self._types
        tokens, width = x.shape
        dev = x.get_device()
        need_tensor(x, types.float, (tokens, width), 'x', dev)
        need_tensor(codes, types.e4m3, (tokens, width), 'codes', dev)
        need_tensor(scales, types.float, (-(-width // 128), tokens), 'scales', dev)
        need_tensor(weights, types.float, (width,), 'weights', dev)
        for name, t in (('residual', residual), ('residual_out', residual_out), ('normed', normed)):
            if t is not None:
                need_tensor(t, types.float, (tokens, width), name, dev)
        self._call(dev, self.lib.qv_norm8, codes.data_ptr(), scales.data_ptr(),
                   None if residual_out is None else residual_out.data_ptr(),
                   None if normed is None else normed.data_ptr(), x.data_ptr(),
                   None if residual is None else residual.data_ptr(), weights.data_ptr(), tokens, width, epsilon)

    def quantize8(self, codes, scales, x):
        """qv_quantize8: e4m3 codes and scales of x itself."""
        types = self._types
        tokens, width = x.shape
        dev = x.get_device()
        need_tensor(x, types.float, (tokens, width), 'x', dev)
        need_tensor(codes, types.e4m3, (tokens, width), 'codes', dev)
        need_tensor(scales, types.float, (-(-width // 128), tokens), 'scales', dev)
        self._call(dev, self.lib.qv_quantize8, codes.data_ptr(), scales.data_ptr(), x.data_ptr(), tokens, width)

    def mm8(self, out, weights, weight_scales, codes, scales):
        """qv_mm8: out [tokens][rows] = codes x weights^T, both e4m3 with a scale for every block of 128."""
        types = self._types
        tokens, width = codes.shape
        rows, blocks, dev = weights.shape[0], -(-width // 128), codes.get_device()
        need_tensor(codes, types.e4m3, (tokens, width), 'codes', dev)
        need_tensor(scales, types.float, (blocks, tokens), 'scales', dev)
        need_tensor(weights, types.e4m3, (rows, width), 'weights', dev)
        need_tensor(weight_scales, types.float, (-(-rows // 128), blocks), 'weight_scales', dev)
        need_tensor(out, types.float, (tokens, rows), 'out', dev)
        self._call(dev, self.lib.qv_mm8, out.data_ptr(), weights.data_ptr(), weight_scales.data_ptr(), codes.data_ptr(),
                   scales.data_ptr(), tokens, width, rows)

    def attention8_workspace(self, device):
        """A new workspace for attention8 at any batch and position: the barrier words in its first 256 bytes
        are zero.  One serves one call at a time; a captured graph keeps one of its own."""
        import torch
        # the split partials of the longest context, which no shorter one exceeds
        need = max(self.lib.qv_attention8_workspace(1, 139263), self.lib.qv_attention8_workspace(1, 64 * 37 - 1))
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:256].zero_()
        return ws

    KEPT_WORKSPACES8 = 16

    def kept_workspace8(self, device):
        """The workspace of the current stream of device number `device`.  The newest KEPT_WORKSPACES8 are kept
        (10 MB each); an older one goes back to torch's allocator, which gives its memory to later work of the
        same stream only."""
        import torch
        which = (device, torch._C._cuda_getCurrentRawStream(device))
        workspace = self._workspaces8.get(which)
        if workspace is None:
            workspace = self._workspaces8[which] = self.attention8_workspace(torch.device('cuda', device))
            while len(self._workspaces8) > self.KEPT_WORKSPACES8:
                self._workspaces8.pop(next(iter(self._workspaces8)), None)
        return workspace

    def attention8(self, out, key_codes, key_scales, value_codes, value_scales, packed, key_tail, value_tail, q_gate,
                   key, value, q_norm, k_norm, batch, position, epsilon=1e-6, workspace=None):
        """qv_attention8: one attention layer for 1..10 new tokens over the 8-bit cache's first `packed`
        positions and the fp16 tail.  Without `workspace`, one that is kept for the current stream is used;
        under graph capture it has to be given (attention8_workspace), since the graph goes on using it."""
        types = self._types
        dev, tail = out.get_device(), key_tail.shape[0]
        need_tensor(out, types.float, (batch, 24, 256), 'out', dev)
        need_tensor(q_gate, types.float, (batch, 24, 512), 'q_gate', dev)
        need_tensor(key, types.float, (batch, 4, 256), 'key', dev)
        need_tensor(value, types.float, (batch, 4, 256), 'value', dev)
        need_tensor(q_norm, types.float, (256,), 'q_norm', dev)
        need_tensor(k_norm, types.float, (256,), 'k_norm', dev)
        need_tensor(key_tail, types.half, (tail, 4, 256), 'key_tail', dev)
        need_tensor(value_tail, types.half, (tail, 4, 256), 'value_tail', dev)
        need_cache8(types, key_codes, key_scales, value_codes, value_scales, packed, dev)
        if workspace is None:
            if self.capturing(dev):
                raise ValueError('attention8 under graph capture needs a workspace of its own (attention8_workspace)')
            workspace = self.kept_workspace8(dev)
        else:
            need_tensor(workspace, types.bytes, workspace.shape, 'workspace', dev)
        self._call(dev, self.lib.qv_attention8, out.data_ptr(), key_codes.data_ptr(), key_scales.data_ptr(),
                   value_codes.data_ptr(), value_scales.data_ptr(), packed, key_tail.data_ptr(), value_tail.data_ptr(), tail,
                   q_gate.data_ptr(), key.data_ptr(), value.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(),
                   batch, position, epsilon, workspace.data_ptr(), workspace.numel())

    def cache8_pack(self, key_codes, key_scales, value_codes, value_scales, key_rows, value_rows, begin, end):
        """qv_cache8_pack: positions [begin, end) of fp16 rows (position r at row r % rows) to int8 codes."""
        types = self._types
        ring, dev = key_rows.shape[0], key_rows.get_device()
        need_cache8(types, key_codes, key_scales, value_codes, value_scales, end, dev)
        need_tensor(key_rows, types.half, (ring, 4, 256), 'key_rows', dev)
        need_tensor(value_rows, types.half, (ring, 4, 256), 'value_rows', dev)
        self._call(dev, self.lib.qv_cache8_pack, key_codes.data_ptr(), key_scales.data_ptr(), value_codes.data_ptr(),
                   value_scales.data_ptr(), key_rows.data_ptr(), value_rows.data_ptr(), begin, end, ring)

    def cache8_unpack(self, key_rows, value_rows, key_codes, key_scales, value_codes, value_scales, begin, end, origin=0):
        """qv_cache8_unpack: positions [begin, end) as fp16 rows, position r at row r - origin."""
        types = self._types
        rows, dev = key_rows.shape[0], key_rows.get_device()
        need_cache8(types, key_codes, key_scales, value_codes, value_scales, end, dev)
        need_tensor(key_rows, types.half, (rows, 4, 256), 'key_rows', dev)
        need_tensor(value_rows, types.half, (rows, 4, 256), 'value_rows', dev)
        if not 0 <= begin - origin <= end - origin <= rows:
            raise ValueError(f'positions [{begin}, {end}) do not fit {rows} rows from position {origin}')
        skip = (begin - origin) * 2048
        self._call(dev, self.lib.qv_cache8_unpack, key_rows.data_ptr() + skip, value_rows.data_ptr() + skip,
                   key_codes.data_ptr(), key_scales.data_ptr(), value_codes.data_ptr(), value_scales.data_ptr(), begin, end)

    def status(self):
        """Synchronise and return the kernel status word (0 = no timeout)."""
        code = self.lib.qv_status()
        if code < 0:
            raise NativeError(self.lib.qv_error().decode('utf-8', errors='replace'))
        return code
