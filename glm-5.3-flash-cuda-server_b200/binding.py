"""ctypes binding of libb200nvfp4.so for tests and benchmarks.

The product is the shared library and its C ABI (include/b200_nvfp4.h); this file only moves
pointers.  torch is used for device memory and streams.  There is no fallback of any kind: if
the library has not been built, or a call returns a non-zero status, an exception is raised.
"""
import ctypes as C
import os
import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get('B200_NVFP4_LIB') or os.path.join(_HERE, 'libb200nvfp4.so')
_lib = None

F32, BF16, I8 = 0, 1, 2
GEMV_MULTI_MAX, GEMV_M_MAX = 8, 8


class WRef(C.Structure):
    _fields_ = [('p', C.c_void_p), ('packed', C.c_void_p), ('scale', C.c_void_p), ('gscale', C.c_void_p)]


class GemvJob(C.Structure):
    _fields_ = [('y', C.c_void_p), ('W', WRef), ('x', C.c_void_p), ('N', C.c_int)]


class Nvfp4Mat(C.Structure):
    _fields_ = [('packed', C.c_void_p), ('scale', C.c_void_p), ('gscale', C.c_void_p)]


class I8RowsC(C.Structure):
    _fields_ = [('q', C.c_void_p), ('scale', C.c_void_p)]


class MoeLayerC(C.Structure):
    _fields_ = [('router_w', WRef), ('router_bias', C.c_void_p), ('experts', C.c_void_p),
                ('shared', C.c_void_p), ('n_expert', C.c_int), ('topk', C.c_int), ('hidden', C.c_int),
                ('inter', C.c_int), ('routed_scale', C.c_float), ('swiglu_limit', C.c_float),
                ('norm_topk', C.c_int)]


class EpStats(C.Structure):
    _fields_ = [('tokens', C.c_int), ('recv_rows', C.c_int), ('sent_remote_rows', C.c_int), ('recv_remote_rows', C.c_int),
                ('local_experts_touched', C.c_int), ('pad', C.c_int), ('dispatch_bytes_out', C.c_ulonglong),
                ('combine_bytes_in', C.c_ulonglong), ('plan_us', C.c_float), ('dispatch_us', C.c_float),
                ('experts_us', C.c_float), ('combine_us', C.c_float), ('total_us', C.c_float), ('pad2', C.c_float)]


class OverlayEntry(C.Structure):
    _fields_ = [('packed', C.c_void_p), ('scale', C.c_void_p), ('gscale', C.c_float), ('N', C.c_int), ('K', C.c_int)]


class B200Error(RuntimeError):
    pass


def lib():
    """The loaded library; raises if it has not been built (python -c 'import __graft_entry__ as g; g.build()')."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise B200Error('libb200nvfp4.so is missing at %s: build it first; there is no CPU fallback' % LIB_PATH)
        L = C.CDLL(LIB_PATH)
        vp, ci, st = C.c_void_p, C.c_int, C.c_size_t
        L.b200_nvfp4_strerror.restype = C.c_char_p; L.b200_nvfp4_strerror.argtypes = [ci]
        L.b200_nvfp4_version.restype = ci
        L.b200_nvfp4_device_status.argtypes = [C.POINTER(C.c_uint), ci]
        L.b200_nvfp4_selftest_bounded_wait.argtypes = [vp]
        L.b200_nvfp4_set_byte_credit.argtypes = [vp, vp]
        L.b200_nvfp4_flush_byte_credit.argtypes = [ci]
        L.b200_nvfp4_gemm.argtypes = [vp, C.POINTER(WRef), vp, ci, ci, ci, ci, vp]
        L.b200_nvfp4_gemv_multi.argtypes = [C.POINTER(GemvJob), ci, ci, ci, ci, vp]
        L.b200_nvfp4_split_workspace_bytes.restype = st; L.b200_nvfp4_split_workspace_bytes.argtypes = [ci, ci]
        L.b200_nvfp4_gemm_ws.argtypes = [vp, C.POINTER(WRef), vp, ci, ci, ci, ci, vp, vp]
        L.b200_nvfp4_gemv_multi_ws.argtypes = [C.POINTER(GemvJob), ci, ci, ci, ci, vp, vp]
        L.b200_nvfp4_gemm_bf16_workspace_bytes.restype = st; L.b200_nvfp4_gemm_bf16_workspace_bytes.argtypes = [ci, ci]
        L.b200_nvfp4_gemm_bf16.argtypes = [vp, C.POINTER(WRef), vp, ci, ci, ci, vp, vp]
        L.b200_nvfp4_quantize_tokens.argtypes = [vp, ci, ci, ci, vp, vp, vp, vp]
        L.b200_nvfp4_gemm_bf16_exact_workspace_bytes.restype = st; L.b200_nvfp4_gemm_bf16_exact_workspace_bytes.argtypes = [ci, ci]
        L.b200_nvfp4_gemm_bf16_exact.argtypes = [vp, C.POINTER(WRef), vp, ci, ci, ci, vp, vp]
        L.b200_dense_mlp_workspace_bytes.restype = st; L.b200_dense_mlp_workspace_bytes.argtypes = [ci, ci, ci]
        L.b200_dense_mlp.argtypes = [vp, C.POINTER(WRef), C.POINTER(WRef), C.POINTER(WRef), ci, ci, C.c_float, vp, vp, ci, vp]
        L.b200_f32_to_bf16.argtypes = [vp, vp, st, vp]
        L.b200_bf16_to_f32.argtypes = [vp, vp, st, vp]
        L.b200_nvfp4_quantize.argtypes = [vp, ci, ci, vp, vp, vp, vp, vp]
        L.b200_nvfp4_dequantize.argtypes = [vp, C.POINTER(Nvfp4Mat), ci, ci, vp]
        L.b200_i8_pitch.restype = st; L.b200_i8_pitch.argtypes = [ci]
        L.b200_i8_quantize.argtypes = [vp, ci, st, ci, ci, vp, vp, vp]
        L.b200_i8_gemm_workspace_bytes.restype = st; L.b200_i8_gemm_workspace_bytes.argtypes = [ci, ci]
        L.b200_i8_gemm.argtypes = [vp, ci, C.POINTER(I8RowsC), vp, ci, st, ci, ci, ci, vp, vp]
        L.b200_token_logprobs.argtypes = [vp, ci, st, ci, ci, vp, ci, vp, vp, ci, vp, vp, vp]
        L.b200_moe_workspace_bytes.restype = st; L.b200_moe_workspace_bytes.argtypes = [C.POINTER(MoeLayerC), ci]
        L.b200_moe_route.argtypes = [vp, C.POINTER(MoeLayerC), vp, vp, vp, ci, vp]
        L.b200_moe_forward.argtypes = [vp, C.POINTER(MoeLayerC), vp, vp, vp, vp, ci, vp]
        L.b200_moe_experts.argtypes = [vp, C.POINTER(MoeLayerC), vp, vp, vp, vp, ci, vp]
        L.b200_moe_forward_static.argtypes = [vp, C.POINTER(MoeLayerC), vp, vp, vp, ci, vp]
        L.b200_moe_static_ws_limit.restype = st
        L.b200_ep_unique_id.argtypes = [vp]
        L.b200_ep_create.argtypes = [C.POINTER(vp), vp, ci, ci, C.POINTER(MoeLayerC), C.POINTER(MoeLayerC), C.POINTER(MoeLayerC), ci]
        L.b200_ep_forward.argtypes = [vp, vp, vp, vp, vp, ci, vp]
        L.b200_ep_last_stats.argtypes = [vp, C.POINTER(EpStats)]
        L.b200_ep_destroy.argtypes = [vp]
        L.b200_overlay_writer_open.argtypes = [C.POINTER(vp), C.c_char_p, C.c_uint64]
        L.b200_overlay_writer_add.argtypes = [vp, C.c_char_p, vp, vp, C.c_float, ci, ci]
        L.b200_overlay_writer_close.argtypes = [vp]
        L.b200_overlay_family.argtypes = [C.c_char_p, C.c_char_p, C.c_char_p]
        L.b200_overlay_open.argtypes = [C.POINTER(vp), C.c_char_p]
        L.b200_overlay_count.argtypes = [vp]
        L.b200_overlay_find.argtypes = [vp, C.c_char_p, C.POINTER(OverlayEntry)]
        L.b200_overlay_close.argtypes = [vp]
        L.b200_moe_prepare.argtypes = [C.POINTER(MoeLayerC)]
        L.b200_moe_release.argtypes = [C.POINTER(MoeLayerC)]
        _lib = L
    return _lib


ENOTIMPL = 6
EXPORTS = ['b200_nvfp4_set_byte_credit', 'b200_nvfp4_flush_byte_credit', 'b200_nvfp4_strerror', 'b200_nvfp4_version', 'b200_nvfp4_device_status', 'b200_nvfp4_selftest_bounded_wait', 'b200_nvfp4_set_option', 'b200_nvfp4_gemm', 'b200_nvfp4_gemv_multi', 'b200_nvfp4_split_workspace_bytes', 'b200_nvfp4_gemm_ws', 'b200_nvfp4_gemv_multi_ws',
           'b200_nvfp4_gemm_bf16_workspace_bytes', 'b200_nvfp4_gemm_bf16', 'b200_nvfp4_quantize_tokens', 'b200_nvfp4_gemm_bf16_exact_workspace_bytes', 'b200_nvfp4_gemm_bf16_exact', 'b200_dense_mlp_workspace_bytes', 'b200_dense_mlp', 'b200_f32_to_bf16', 'b200_bf16_to_f32', 'b200_nvfp4_quantize', 'b200_nvfp4_dequantize',
           'b200_i8_pitch', 'b200_i8_quantize', 'b200_i8_gemm_workspace_bytes', 'b200_i8_gemm', 'b200_token_logprobs',
           'b200_moe_workspace_bytes', 'b200_moe_route', 'b200_moe_forward', 'b200_moe_experts',
           'b200_moe_forward_static', 'b200_moe_static_ws_limit', 'b200_moe_prepare', 'b200_moe_release',
           'b200_overlay_writer_open', 'b200_overlay_writer_add', 'b200_overlay_writer_close', 'b200_overlay_family',
           'b200_overlay_open', 'b200_overlay_count', 'b200_overlay_find', 'b200_overlay_close',
           'b200_ep_unique_id', 'b200_ep_create', 'b200_ep_forward', 'b200_ep_last_stats', 'b200_ep_destroy']


def check(rc, what):
    if rc != 0:
        raise B200Error('%s failed: %s (%d)' % (what, lib().b200_nvfp4_strerror(rc).decode(), rc))


def device_status(clear=False):
    """0 unless a bounded wait inside a kernel ever ran out (synchronises the device)."""
    v = C.c_uint(0)
    check(lib().b200_nvfp4_device_status(C.byref(v), 1 if clear else 0), 'b200_nvfp4_device_status')
    return v.value


OPT_STABLE_WEIGHTS = 1
OPT_PREFILL_FP4 = 2


def set_option(option, value):
    check(lib().b200_nvfp4_set_option(int(option), int(value)), 'b200_nvfp4_set_option')


def stream_ptr(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _stream(stream):
    """The cudaStream_t as an int (an argument of type c_void_p takes one without an object in between).
    torch.cuda.current_stream() builds a Stream object (3.4 us, as long as a whole launch); the raw handle of the
    same stream takes 0.1 us."""
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _empty(stream, shape, dtype, device):
    """What a call on `stream` allocates itself.  The memory is that stream's: a block of the current stream's could be one that a kernel
    pending there still uses.  It is not given away either before the current stream, whose owner gets the tensor, is done with it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    here = torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(here)
    return t


def _ptr(t):
    return t.data_ptr() if t is not None else None


class Nvfp4Weight:
    """An NVFP4 triple resident on the device (packed u8 [N,K/2], scale u8 [N,K/16], gscale f32 [1])."""

    def __init__(self, packed, scale, gscale, device='cuda'):
        to = lambda a, dt: (torch.from_numpy(np.ascontiguousarray(a)) if isinstance(a, np.ndarray) else a).to(device=device, dtype=dt).contiguous()
        self.packed, self.scale, self.gscale = to(packed, torch.uint8), to(scale, torch.uint8), to(gscale, torch.float32)
        self.N, self.K = self.packed.shape[0], self.packed.shape[1] * 2

    def wref(self):
        return WRef(None, self.packed.data_ptr(), self.scale.data_ptr(), self.gscale.data_ptr())

    def mat(self):
        return Nvfp4Mat(self.packed.data_ptr(), self.scale.data_ptr(), self.gscale.data_ptr())

    def numpy(self):
        return self.packed.cpu().numpy(), self.scale.cpu().numpy(), self.gscale.cpu().numpy()

    @property
    def nbytes(self):
        return self.packed.numel() + self.scale.numel() + 4


def split_workspace(M, K, device, stream=None):
    """Scratch for gemm(..., ws=) / gemv_multi(..., ws=): the pre-split activation images."""
    return _empty(stream, lib().b200_nvfp4_split_workspace_bytes(M, K), torch.uint8, device)


def gemm(W, x, y=None, dtype=BF16, stream=None, ws=None):
    """y[M,N] = x[M,K] . W^T.  W: Nvfp4Weight, or a bf16/f32 torch tensor [N,K].  ws: split_workspace(M, K)."""
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    M, K = x2.shape
    if isinstance(W, Nvfp4Weight):
        N, ref = W.N, W.wref()
        assert W.K == K
    else:
        N, ref = W.shape[0], WRef(W.data_ptr(), None, None, None)
        dtype = F32 if W.dtype == torch.float32 else BF16
    if y is None:
        y = _empty(stream, (M, N), torch.float32, x.device)
    if ws is not None:
        check(lib().b200_nvfp4_gemm_ws(_ptr(y), C.byref(ref), _ptr(x2), M, N, K, dtype, _ptr(ws), _stream(stream)), 'b200_nvfp4_gemm_ws')
    else:
        check(lib().b200_nvfp4_gemm(_ptr(y), C.byref(ref), _ptr(x2), M, N, K, dtype, _stream(stream)), 'b200_nvfp4_gemm')
    return y if x.dim() == 2 else y[0]


def gemm_bf16_workspace(M, K, device, stream=None):
    return _empty(stream, lib().b200_nvfp4_gemm_bf16_workspace_bytes(M, K), torch.uint8, device)


def gemm_bf16(W, x_bf16, y=None, ws=None, stream=None):
    """The wide GEMM: y[M,N] f32 = x[M,K] bf16 . W^T with the activations quantised to NVFP4 per token."""
    M, K = x_bf16.shape
    assert W.K == K and x_bf16.dtype == torch.bfloat16
    if y is None:
        y = _empty(stream, (M, W.N), torch.float32, x_bf16.device)
    if ws is None:
        ws = gemm_bf16_workspace(M, K, x_bf16.device, stream)
    ref = W.wref()
    check(lib().b200_nvfp4_gemm_bf16(_ptr(y), C.byref(ref), _ptr(x_bf16), M, W.N, K, _ptr(ws), _stream(stream)), 'b200_nvfp4_gemm_bf16')
    return y


def gemm_bf16_exact(W, x_bf16, y=None, ws=None, stream=None):
    """The exact wide GEMM: y[M,N] f32 = x[M,K] bf16 . W^T, weights dequantised to fp16 in the kernel."""
    M, K = x_bf16.shape
    assert W.K == K and x_bf16.dtype == torch.bfloat16
    if y is None:
        y = _empty(stream, (M, W.N), torch.float32, x_bf16.device)
    if ws is None:
        ws = _empty(stream, lib().b200_nvfp4_gemm_bf16_exact_workspace_bytes(M, K), torch.uint8, x_bf16.device)
    ref = W.wref()
    check(lib().b200_nvfp4_gemm_bf16_exact(_ptr(y), C.byref(ref), _ptr(x_bf16), M, W.N, K, _ptr(ws), _stream(stream)), 'b200_nvfp4_gemm_bf16_exact')
    return y


def quantize_tokens(x, stream=None):
    """Per-token NVFP4 quantisation of x [M,K] (bf16 or f32): packed [M,K/2], scale [M,K/16] (returned
    row-major; the library writes it step-major), gs [M]."""
    M, K = x.shape
    dev = x.device
    packed = _empty(stream, (M, K // 2), torch.uint8, dev)
    sfb = _empty(stream, (K // 256, M, 16), torch.uint8, dev)
    gs = _empty(stream, (M,), torch.float32, dev)
    scale = _empty(stream, (M, K // 16), torch.uint8, dev)
    check(lib().b200_nvfp4_quantize_tokens(_ptr(x), 1 if x.dtype == torch.float32 else 0, M, K, _ptr(packed), _ptr(sfb), _ptr(gs),
                                           _stream(stream)), 'b200_nvfp4_quantize_tokens')
    with torch.cuda.stream(stream):                     # behind the kernel
        scale.view(M, K // 256, 16).copy_(sfb.permute(1, 0, 2))
    return packed, scale, gs


def dense_mlp_workspace(M, hidden, inter, device, stream=None):
    return _empty(stream, lib().b200_dense_mlp_workspace_bytes(M, hidden, inter), torch.uint8, device)


def dense_mlp(x, gate, up, down, limit=10.0, y=None, ws=None, stream=None):
    """y = down . (silu(min(gate.x, limit)) * clamp(up.x, -limit, limit)); x [M, hidden] f32."""
    M, H = x.shape
    I = gate.N
    if y is None:
        y = _empty(stream, (M, H), torch.float32, x.device)
    if ws is None:
        ws = dense_mlp_workspace(M, H, I, x.device, stream)
    g, u, d = gate.wref(), up.wref(), down.wref()
    check(lib().b200_dense_mlp(_ptr(x), C.byref(g), C.byref(u), C.byref(d), H, I, float(limit), _ptr(y), _ptr(ws), M, _stream(stream)),
          'b200_dense_mlp')
    return y


def gemv(W, x, y=None, stream=None):
    return gemm(W, x, y, stream=stream)


def make_jobs(weights, xs, ys):
    arr = (GemvJob * len(weights))()
    for i, (W, x, y) in enumerate(zip(weights, xs, ys)):
        arr[i] = GemvJob(y.data_ptr(), W.wref(), x.data_ptr(), W.N)
    return arr


def gemv_multi(weights, xs, M=1, ys=None, stream=None, jobs=None, ws=None):
    """Fused group: weights share K; xs is one tensor [M,K] (shared) or a list (one per job)."""
    if not isinstance(xs, (list, tuple)):
        xs = [xs] * len(weights)
    if ys is None:
        ys = [_empty(stream, (M, W.N), torch.float32, xs[0].device) for W in weights]
    if jobs is None:
        jobs = make_jobs(weights, xs, ys)
    if ws is not None:
        check(lib().b200_nvfp4_gemv_multi_ws(jobs, len(weights), M, weights[0].K, BF16, _ptr(ws), _stream(stream)), 'b200_nvfp4_gemv_multi_ws')
    else:
        check(lib().b200_nvfp4_gemv_multi(jobs, len(weights), M, weights[0].K, BF16, _stream(stream)), 'b200_nvfp4_gemv_multi')
    return ys


def f32_to_bf16(src, stream=None):
    dst = _empty(stream, src.shape, torch.bfloat16, src.device)
    check(lib().b200_f32_to_bf16(_ptr(dst), _ptr(src), src.numel(), _stream(stream)), 'b200_f32_to_bf16')
    return dst


def bf16_to_f32(src, stream=None):
    dst = _empty(stream, src.shape, torch.float32, src.device)
    check(lib().b200_bf16_to_f32(_ptr(dst), _ptr(src), src.numel(), _stream(stream)), 'b200_bf16_to_f32')
    return dst


def quantize(w_bf16, gscale_in=None, out=None, stream=None):
    """bf16 [N,K] device tensor -> Nvfp4Weight, bit-exact with the reference quantiser."""
    N, K = w_bf16.shape
    dev = w_bf16.device
    if out is None:
        out = Nvfp4Weight(_empty(stream, (N, K // 2), torch.uint8, dev), _empty(stream, (N, K // 16), torch.uint8, dev),
                          _empty(stream, (1,), torch.float32, dev), device=dev)
    check(lib().b200_nvfp4_quantize(_ptr(w_bf16), N, K, _ptr(out.packed), _ptr(out.scale), _ptr(out.gscale),
                                    _ptr(gscale_in), _stream(stream)), 'b200_nvfp4_quantize')
    return out


def dequantize(W, stream=None):
    out = _empty(stream, (W.N, W.K), torch.float32, W.packed.device)
    m = W.mat()
    check(lib().b200_nvfp4_dequantize(_ptr(out), C.byref(m), W.N, W.K, _stream(stream)), 'b200_nvfp4_dequantize')
    return out


_DTYPE = {torch.float32: F32, torch.bfloat16: BF16}


def _want(ok, what):
    if not ok:
        raise B200Error(what)


def _device(*tensors):
    """Kernels run on the current device's stream: every tensor has to lie there."""
    devs = [t.get_device() for t in tensors]            # -1: not on a GPU
    if min(devs) < 0 or devs.count(torch._C._cuda_getDevice()) != len(devs):
        raise B200Error('tensors have to be on the current CUDA device')


def _strided_rows(x, what):
    """(dtype code, rows, columns, row stride) of a 2-d f32 or bf16 tensor whose rows are contiguous and do not overlap."""
    dt, shape = _DTYPE.get(x.dtype), x.shape
    if dt is None or len(shape) != 2 or shape[0] < 1 or shape[1] < 1:
        raise B200Error(what + ' has to be a non-empty 2-d f32 or bf16 tensor')
    M, K = shape
    if x.is_contiguous():
        return dt, M, K, K
    ld, one = x.stride()
    if M == 1:
        ld = K
    if (one != 1 and K != 1) or ld < K:
        raise B200Error(what + ' has to have contiguous rows')
    return dt, M, K, ld


class I8Rows:
    """Rows of 8-bit integers, a scale per row: q int8 [rows, pitch] (pitch: K rounded up to 32), scale f32 [rows]."""

    def __init__(self, q, scale, K):
        _want(K >= 1 and q.dim() == 2 and q.dtype == torch.int8 and q.is_contiguous() and q.shape[1] == (K + 31) // 32 * 32,
              'q has to be contiguous int8 [rows, K rounded up to 32]')
        _want(scale.dtype == torch.float32 and scale.is_contiguous() and scale.shape == (q.shape[0],), 'scale has to be contiguous f32 [rows]')
        _device(q, scale)
        self._q, self._scale, self.N, self.K, self.dev = q, scale, q.shape[0], K, q.get_device()
        self.c = I8RowsC(q.data_ptr(), scale.data_ptr())
        self.ref, self.addr = C.byref(self.c), C.addressof(self.c)

    # what `c` points to
    q = property(lambda self: self._q)
    scale = property(lambda self: self._scale)

    @classmethod
    def empty(cls, rows, K, device, stream=None):
        _want(rows >= 1 and K >= 1, 'rows and K have to be positive')
        return cls(_empty(stream, (rows, (K + 31) // 32 * 32), torch.int8, device), _empty(stream, (rows,), torch.float32, device), K)

    @property
    def nbytes(self):
        return self.q.numel() + 4 * self.N


def i8_quantize(x, out=None, stream=None):
    """x [rows, K] (f32 or bf16) -> I8Rows, weights (a scale per output channel) and activations (per token) alike."""
    dt, M, K, ld = _strided_rows(x, 'x')
    if out is None:
        _device(x)
        out = I8Rows.empty(M, K, x.device, stream)
    if out.N != M or out.K != K:
        raise B200Error('out has to be I8Rows of the size of x')
    dev = torch._C._cuda_getDevice()
    if x.get_device() != dev or out.dev != dev:
        raise B200Error('tensors have to be on the current CUDA device')
    rc = lib().b200_i8_quantize(x.data_ptr(), dt, ld, M, K, out.c.q, out.c.scale, _stream(stream))
    if rc:
        check(rc, 'b200_i8_quantize')
    return out


def i8_gemm_workspace(M, K, device, stream=None):
    """Scratch for i8_gemm on f32 or bf16 activations: their 8-bit rows."""
    return _empty(stream, lib().b200_i8_gemm_workspace_bytes(M, K), torch.uint8, device)


def i8_gemm(W, x, y=None, ws=None, dtype=torch.float32, stream=None):
    """y[M,N] (f32 or bf16) = x[M,K] . W^T in 8-bit integers.  W: I8Rows; x: I8Rows, or f32 / bf16 rows, which are quantised
    within the call, into ws (i8_gemm_workspace(M, K))."""
    dev = torch._C._cuda_getDevice()
    if type(x) is I8Rows:
        M, K, xp, dx, ld, wp, here = x.N, x.K, x.addr, I8, 0, None, x.dev          # x itself holds what xp points to: it stays bound
    else:
        dx, M, K, ld = _strided_rows(x, 'x')
        xp, here = x.data_ptr(), x.get_device()
        if ws is None:
            ws = i8_gemm_workspace(M, K, x.device, stream)
        if not ws.is_contiguous() or ws.nbytes < (M * ((K + 31) & ~31) + 255 & ~255) + (4 * M + 255 & ~255):
            raise B200Error('ws is smaller than i8_gemm_workspace(M, K)')
        wp = ws.data_ptr()
        if ws.get_device() != here:
            raise B200Error('tensors have to be on the current CUDA device')
    N = W.N
    if W.K != K:
        raise B200Error('W and x have to share K')
    if y is None:
        y = _empty(stream, (M, N), dtype, W.q.device)
    dy, shape = _DTYPE.get(y.dtype), y.shape
    if dy is None or len(shape) != 2 or shape[0] != M or shape[1] != N or not y.is_contiguous():
        raise B200Error('y has to be contiguous f32 or bf16 [M, N]')
    if here != dev or W.dev != dev or y.get_device() != dev:
        raise B200Error('tensors have to be on the current CUDA device')
    rc = lib().b200_i8_gemm(y.data_ptr(), dy, W.ref, xp, dx, ld, M, N, K, wp, stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, 'b200_i8_gemm')
    return y


LOGPROBS_TOP_MAX = 32


class LogprobsOut(tuple):
    """(logprobs [M, G], entropy [M], top_ids [M, top], top_logprobs [M, top]), checked once: token_logprobs_out."""

    @classmethod
    def of(cls, tensors, M, G, top):
        lp, ent, ids, tlp = tensors
        if (lp.shape != (M, G) or ent.shape != (M,) or ids.shape != (M, top) or tlp.shape != (M, top) or ids.dtype != torch.int32 or
                not (lp.dtype == ent.dtype == tlp.dtype == torch.float32) or
                not (lp.is_contiguous() and ent.is_contiguous() and ids.is_contiguous() and tlp.is_contiguous())):
            raise B200Error('out has to be token_logprobs_out(tokens, top)')
        _device(lp, ent, ids, tlp)
        self = cls(tensors)
        self.size, self.dev = (M, G, top), lp.get_device()
        self.ptrs = lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), tlp.data_ptr()
        return self


def token_logprobs_out(tokens, top, stream=None):
    """Output buffers of token_logprobs for these tokens."""
    _want(tokens.dim() == 2 and top >= 0, 'tokens has to be [M, G], top not negative')
    M, G = tokens.shape
    new = lambda shape, dtype=torch.float32: _empty(stream, shape, dtype, tokens.device)
    return LogprobsOut.of((new((M, G)), new((M,)), new((M, top), torch.int32), new((M, top))), M, G, top)


def token_logprobs(logits, tokens, top=0, out=None, stream=None):
    """ln p of the given tokens (tokens int32 [M, G]; negative: none, 0), the entropy in nats, and the `top` likeliest tokens of every
    row of logits [M, V] (f32 or bf16): (logprobs [M, G], entropy [M], top_ids [M, top], top_logprobs [M, top])."""
    dt, M, V, ld = _strided_rows(logits, 'logits')
    shape = tokens.shape
    if tokens.dtype != torch.int32 or len(shape) != 2 or shape[0] != M or not tokens.is_contiguous():
        raise B200Error('tokens has to be contiguous int32 [M, G]')
    G = shape[1]
    if out is None:
        out = token_logprobs_out(tokens, top, stream)
    elif type(out) is not LogprobsOut or out.size != (M, G, top):
        out = LogprobsOut.of(out, M, G, top)
    dev = torch._C._cuda_getDevice()
    if logits.get_device() != dev or tokens.get_device() != dev or out.dev != dev:
        raise B200Error('tensors have to be on the current CUDA device')
    lp, ent, ids, tlp = out.ptrs
    rc = lib().b200_token_logprobs(logits.data_ptr(), dt, ld, M, V, tokens.data_ptr(), G, lp, ent, top, ids, tlp, _stream(stream))
    if rc:
        check(rc, 'b200_token_logprobs')
    return out


class MoeLayer:
    """Device-side description of one MoE layer: router, bias, expert pointer tables."""

    def __init__(self, router_bf16, bias, experts, shared, topk, hidden, inter, routed_scale=2.5,
                 swiglu_limit=10.0, norm_topk=True):
        """experts: list of (gate, up, down) Nvfp4Weight; shared: one such triple or None."""
        dev = router_bf16.device
        self.router, self.bias, self.experts, self.shared = router_bf16, bias, experts, shared
        flat = []
        for g, u, d in experts:
            for w in (g, u, d):
                flat += [w.packed.data_ptr(), w.scale.data_ptr(), w.gscale.data_ptr()]
        self.table = torch.tensor(flat, dtype=torch.int64).to(dev)
        self.shared_table = None
        if shared is not None:
            fl = []
            for w in shared:
                fl += [w.packed.data_ptr(), w.scale.data_ptr(), w.gscale.data_ptr()]
            self.shared_table = torch.tensor(fl, dtype=torch.int64).to(dev)
        self.c = MoeLayerC(WRef(router_bf16.data_ptr(), None, None, None), bias.data_ptr(), self.table.data_ptr(),
                           self.shared_table.data_ptr() if shared is not None else None,
                           len(experts), topk, hidden, inter, routed_scale, swiglu_limit, 1 if norm_topk else 0)
        self.topk, self.hidden, self.inter, self.n_expert = topk, hidden, inter, len(experts)
        self._ws = {}

    def workspace(self, M):
        if M not in self._ws:
            n = lib().b200_moe_workspace_bytes(C.byref(self.c), M)
            self._ws[M] = torch.empty(n, dtype=torch.uint8, device=self.router.device)
            # kept for calls on any stream: whatever used this memory before has to be done with it
            if self._ws[M].is_cuda and not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        return self._ws[M]


def moe_route(layer, x, stream=None):
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    M = x2.shape[0]
    sel = _empty(stream, (M, layer.topk), torch.int32, x.device)
    wts = _empty(stream, (M, layer.topk), torch.float32, x.device)
    logits = _empty(stream, (M, layer.n_expert), torch.float32, x.device)
    check(lib().b200_moe_route(_ptr(x2), C.byref(layer.c), _ptr(sel), _ptr(wts), _ptr(logits), M, _stream(stream)), 'b200_moe_route')
    return sel, wts, logits


def moe_forward(layer, x, y=None, sel=None, wts=None, stream=None):
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    M = x2.shape[0]
    dev = x.device
    y = _empty(stream, (M, layer.hidden), torch.float32, dev) if y is None else y
    sel = _empty(stream, (M, layer.topk), torch.int32, dev) if sel is None else sel
    wts = _empty(stream, (M, layer.topk), torch.float32, dev) if wts is None else wts
    ws = layer.workspace(M)
    check(lib().b200_moe_forward(_ptr(x2), C.byref(layer.c), _ptr(y), _ptr(sel), _ptr(wts), _ptr(ws), M, _stream(stream)), 'b200_moe_forward')
    return y, sel, wts


def moe_prepare(layer):
    """Build the layer's TMA descriptors so that batches of up to 8 tokens run on the tensor-core
    kernels.  Returns False when the geometry does not suit them (the layer keeps the CUDA-core path)."""
    rc = lib().b200_moe_prepare(C.byref(layer.c))
    if rc == ENOTIMPL:
        return False
    check(rc, 'b200_moe_prepare')
    return True


def moe_release(layer):
    check(lib().b200_moe_release(C.byref(layer.c)), 'b200_moe_release')


def moe_experts(layer, x, sel, wts, y=None, stream=None):
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    M = x2.shape[0]
    y = _empty(stream, (M, layer.hidden), torch.float32, x.device) if y is None else y
    ws = layer.workspace(M)
    check(lib().b200_moe_experts(_ptr(x2), C.byref(layer.c), _ptr(y), _ptr(sel), _ptr(wts), _ptr(ws), M, _stream(stream)), 'b200_moe_experts')
    return y


def moe_forward_static(layer, x, y=None, sel=None, wts=None, stream=None):
    """moe_forward through the library's built-in scratch (no workspace tensor is created here)."""
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    M = x2.shape[0]
    dev = x.device
    y = _empty(stream, (M, layer.hidden), torch.float32, dev) if y is None else y
    sel = _empty(stream, (M, layer.topk), torch.int32, dev) if sel is None else sel
    wts = _empty(stream, (M, layer.topk), torch.float32, dev) if wts is None else wts
    check(lib().b200_moe_forward_static(_ptr(x2), C.byref(layer.c), _ptr(y), _ptr(sel), _ptr(wts), M, _stream(stream)),
          'b200_moe_forward_static')
    return y, sel, wts


def ep_unique_id():
    """128 bytes that identify a new NCCL communicator (call on one rank, hand to all)."""
    buf = C.create_string_buffer(128)
    check(lib().b200_ep_unique_id(buf), 'b200_ep_unique_id')
    return buf.raw


class EpContext:
    """An expert-parallel layer context of the library (b200_ep_*): this object only holds the handle."""

    def __init__(self, router, local, shared, rank, world, max_tokens, unique_id=None):
        self.h = C.c_void_p(0)
        self.router, self.local, self.shared = router, local, shared      # keep the tables alive
        idbuf = C.create_string_buffer(unique_id, 128) if unique_id is not None else None
        check(lib().b200_ep_create(C.byref(self.h), idbuf, rank, world, C.byref(router.c), C.byref(local.c),
                                   C.byref(shared.c) if shared is not None else None, max_tokens), 'b200_ep_create')

    def forward(self, x, y=None, sel=None, wts=None, stream=None):
        T, dev = x.shape[0], x.device
        y = _empty(stream, (T, self.router.hidden), torch.float32, dev) if y is None else y
        sel = _empty(stream, (T, self.router.topk), torch.int32, dev) if sel is None else sel
        wts = _empty(stream, (T, self.router.topk), torch.float32, dev) if wts is None else wts
        check(lib().b200_ep_forward(self.h, _ptr(x), _ptr(y), _ptr(sel), _ptr(wts), T, _stream(stream)), 'b200_ep_forward')
        return y, sel, wts

    def stats(self):
        st = EpStats()
        check(lib().b200_ep_last_stats(self.h, C.byref(st)), 'b200_ep_last_stats')
        return {k: getattr(st, k) for k, _ in EpStats._fields_ if not k.startswith('pad')}

    def close(self):
        if self.h:
            check(lib().b200_ep_destroy(self.h), 'b200_ep_destroy')
            self.h = C.c_void_p(0)


class OverlayWriter:
    """safetensors overlay of NVFP4 triples, byte-compatible with the reference's requant tool."""

    def __init__(self, directory, shard_bytes=0):
        self.h = C.c_void_p(0)
        check(lib().b200_overlay_writer_open(C.byref(self.h), directory.encode(), shard_bytes), 'b200_overlay_writer_open')

    def add(self, name, packed, scale, gscale):
        """packed u8 [N,K/2], scale u8 [N,K/16]: numpy arrays (host); gscale: float."""
        packed = np.ascontiguousarray(packed, np.uint8); scale = np.ascontiguousarray(scale, np.uint8)
        N, K = packed.shape[0], packed.shape[1] * 2
        check(lib().b200_overlay_writer_add(self.h, name.encode(), packed.ctypes.data_as(C.c_void_p), scale.ctypes.data_as(C.c_void_p),
                                            C.c_float(float(gscale)), N, K), 'b200_overlay_writer_add')

    def close(self):
        check(lib().b200_overlay_writer_close(self.h), 'b200_overlay_writer_close')
        self.h = C.c_void_p(0)


def overlay_family(arch, families, name):
    return lib().b200_overlay_family(arch.encode(), families.encode() if families else None, name.encode())


class Overlay:
    """Reader: maps an overlay directory; triple(name) -> (packed, scale, gscale) numpy copies."""

    def __init__(self, directory):
        self.h = C.c_void_p(0)
        check(lib().b200_overlay_open(C.byref(self.h), directory.encode()), 'b200_overlay_open')

    def __len__(self):
        return lib().b200_overlay_count(self.h)

    def triple(self, name):
        e = OverlayEntry()
        check(lib().b200_overlay_find(self.h, name.encode(), C.byref(e)), 'b200_overlay_find')
        p = np.ctypeslib.as_array(C.cast(e.packed, C.POINTER(C.c_uint8)), shape=(e.N, e.K // 2)).copy()
        s = np.ctypeslib.as_array(C.cast(e.scale, C.POINTER(C.c_uint8)), shape=(e.N, e.K // 16)).copy()
        return p, s, np.array([e.gscale], np.float32), (e.packed % 16 == 0 and e.scale % 16 == 0)

    def close(self):
        check(lib().b200_overlay_close(self.h), 'b200_overlay_close')
        self.h = C.c_void_p(0)


CREDIT_FN = C.CFUNCTYPE(None, C.c_int, C.c_double, C.c_void_p)


class ByteCredit:
    """Collects the weight bytes the library reports per launch site (b200_nvfp4_set_byte_credit)."""

    def __init__(self):
        self.by_kind = {}
        self._cb = CREDIT_FN(lambda kind, nbytes, user: self.by_kind.__setitem__(kind, self.by_kind.get(kind, 0.0) + nbytes))

    def __enter__(self):
        check(lib().b200_nvfp4_set_byte_credit(C.cast(self._cb, C.c_void_p), None), 'b200_nvfp4_set_byte_credit')
        return self

    def flush(self, credit=True):
        check(lib().b200_nvfp4_flush_byte_credit(1 if credit else 0), 'b200_nvfp4_flush_byte_credit')

    def __exit__(self, *a):
        check(lib().b200_nvfp4_set_byte_credit(None, None), 'b200_nvfp4_set_byte_credit')
