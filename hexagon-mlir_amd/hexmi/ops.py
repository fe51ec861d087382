"""Tensor-in / tensor-out operators over libhexmi.so.

Every operator is registered as a PyTorch custom op (`torch.ops.hexmi.*`,
CUDA/HIP dispatch key only) whose implementation hands device pointers and the
current HIP stream to the C ABI. The public functions below add what the
reference's launcher does around a kernel: host tensors are accepted, staged
to the GPU, and results are written back into the caller's `out` tensor in
place (qcom_hexagon_backend/backend/triton_hexagon_launcher.py:716-728 copies
device results back into the tensors the user passed).

There is no CPU implementation: without a GPU or without libhexmi.so these
functions raise.
"""
import ctypes
import math
import warnings

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.int8: _lib.I8}


def _dt(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError("hexmi: unsupported dtype %s" % t.dtype) from None


_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_RAW_DEVICE = getattr(torch._C, "_cuda_getDevice", None)


def _stream():
    """The current device's current HIP stream as an integer handle (the raw getters skip building a
    torch.cuda.Stream object per call, which costs more than a ctypes call)."""
    if _RAW_STREAM is not None and _RAW_DEVICE is not None:
        return _RAW_STREAM(_RAW_DEVICE())
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


class _NoSwitch:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_SWITCH = _NoSwitch()


def _on(device):
    """Context that makes `device` current for the launch; free when it already is (the usual case: entering
    torch.cuda.device() costs more than the shortest kernels here run)."""
    if device.index is None or device.index == (_RAW_DEVICE() if _RAW_DEVICE is not None
                                                else torch.cuda.current_device()):
        return _NO_SWITCH
    return torch.cuda.device(device)


# --------------------------------------------------------------------------
# custom-op registration (schema: inputs..., Tensor(a!) out) -> ()
# --------------------------------------------------------------------------
_LIBDEF = torch.library.Library("hexmi", "DEF")
_LIBDEF.define("softmax(Tensor x, Tensor(a!) out) -> ()")
_LIBDEF.define("rms_norm(Tensor x, Tensor? weight, float eps, Tensor(a!) out) -> ()")
_LIBDEF.define("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, Tensor(a!) out, "
               "Tensor(b!)? mean, Tensor(c!)? rstd) -> ()")
_LIBDEF.define("matmul(Tensor a, Tensor b, bool trans_b, Tensor(a!) out) -> ()")
_LIBDEF.define("linear(Tensor a, Tensor b, Tensor? bias, Tensor? residual, bool trans_b, Tensor(a!) out) -> ()")
_LIBDEF.define("add_matmul_softmax(Tensor x, Tensor y, Tensor z, Tensor(a!) out) -> ()")
_LIBDEF.define("w8a16_matmul(Tensor a, Tensor w, Tensor scales, Tensor(a!) out) -> ()")
_LIBDEF.define("dequant_w8(Tensor w, Tensor scales, Tensor(a!) out) -> ()")
_LIBDEF.define("pack_w8(Tensor w, Tensor(a!) out) -> ()")
_LIBDEF.define("w8a16_matmul_packed(Tensor a, Tensor wp, Tensor scales, Tensor(a!) out) -> ()")
_LIBDEF.define("flash_attention(Tensor q, Tensor k, Tensor v, float sm_scale, bool causal, Tensor(a!) out) -> ()")
_LIBDEF.define("unary(int op, Tensor x, Tensor(a!) out) -> ()")
_LIBDEF.define("binary(int op, Tensor a, Tensor b, Tensor(a!) out) -> ()")
_LIBDEF.define("block_sum(Tensor x, int block, Tensor(a!) out) -> ()")
_LIBDEF.define("rope(Tensor x, float theta, Tensor(a!) out) -> ()")
_LIBDEF.define("attention(Tensor q, Tensor k, Tensor v, Tensor? mask, float sm_scale, Tensor(a!) out) -> ()")
_LIBDEF.define("qk_norm_rope(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor? inv_freq, Tensor? positions, float eps, "
               "str pairs, Tensor(a!) q_out, Tensor(b!)? k_out) -> ()")
_LIBDEF.define("paged_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor lengths, "
               "Tensor? starts, Tensor? k_weight, Tensor? inv_freq, float eps, str pairs, Tensor? q, Tensor? q_weight, "
               "Tensor(c!)? q_out) -> ()")
_LIBDEF.define("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor lengths, Tensor? starts, "
               "float sm_scale, Tensor? shared_pages, Tensor(a!) out) -> ()")


def _row_workspace(rows, cols, block_cols, x):
    """Scratch for the row operators' split form (rows cut into column blocks that several workgroups reduce): the
    library says how much the shape takes, 0 when its single-pass kernels run anyway."""
    need = _lib.lib().hexmi_row_workspace(rows, cols, block_cols, _dt(x))
    return (torch.empty(need, dtype=torch.uint8, device=x.device), need) if need else (None, 0)


def _row_geometry(x, out, rows, cols):
    """(rows, cols, ld_x, ld_out): 2-D tensors whose rows are contiguous may be strided views (ld = row stride);
    anything else is contiguous with rows and cols given."""
    if rows is None:
        rows, cols = x.shape
        return rows, cols, x.stride(0), out.stride(0)
    return rows, cols, cols, cols


def _softmax_impl(x, out, rows=None, cols=None, block_cols=0):
    """x, out: [rows, cols]; or contiguous tensors of any rank with rows and cols given (no view objects built)."""
    rows, cols, ldx, ldo = _row_geometry(x, out, rows, cols)
    with _on(x.device):
        ws, need = _row_workspace(rows, cols, block_cols, x)
        _lib.check(_lib.lib().hexmi_softmax_ws(_p(x), _p(out), rows, cols, ldx, ldo, block_cols, _dt(x), _p(ws), need,
                                               _stream()), "hexmi_softmax_ws")


def _rms_norm_impl(x, weight, eps, out, rows=None, cols=None, block_cols=0):
    rows, cols, ldx, ldo = _row_geometry(x, out, rows, cols)
    with _on(x.device):
        ws, need = _row_workspace(rows, cols, block_cols, x)
        _lib.check(_lib.lib().hexmi_rms_norm_ws(_p(x), _p(weight), _p(out), rows, cols, ldx, ldo, eps, block_cols,
                                                _dt(x), _p(ws), need, _stream()), "hexmi_rms_norm_ws")


def _layer_norm_impl(x, weight, bias, eps, out, mean, rstd, rows=None, cols=None, block_cols=0):
    rows, cols, ldx, ldo = _row_geometry(x, out, rows, cols)
    with _on(x.device):
        ws, need = _row_workspace(rows, cols, block_cols, x)
        _lib.check(_lib.lib().hexmi_layer_norm_ws(_p(x), _p(weight), _p(bias), _p(out), _p(mean), _p(rstd), rows, cols,
                                                  ldx, ldo, eps, block_cols, _dt(x), _p(ws), need, _stream()),
                   "hexmi_layer_norm_ws")


def _matmul_impl(a, b, trans_b, out):
    _linear_impl(a, b, None, None, trans_b, out)


def _linear_impl(a, b, bias, residual, trans_b, out):
    M, K = a.shape
    N = b.shape[0] if trans_b else b.shape[1]
    with _on(a.device):
        # few tiles over a long K: several workgroups share a tile when the library is handed scratch for their fp32 sums
        need = (_lib.lib().hexmi_gemm_workspace(M, N, K, _dt(a), 1 if trans_b else 0)
                if K >= _lib.GEMM_ONE_LAUNCH_K and M * N <= 1 << 20 else 0)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
        _lib.check(_lib.lib().hexmi_gemm_ws(M, N, K, _p(a), a.stride(0), _p(b), b.stride(0), _p(out), out.stride(0),
                                            _p(bias), _p(residual), residual.stride(0) if residual is not None else 0,
                                            _dt(a), _dt(out), 1 if trans_b else 0, _p(ws), need, _stream()), "hexmi_gemm_ws")


def _add_matmul_softmax_impl(x, y, z, out):
    M, K = x.shape
    N = z.shape[1]
    with _on(x.device):
        _lib.check(_lib.lib().hexmi_add_matmul_softmax(M, N, K, _p(x), x.stride(0), _p(y), y.stride(0), _p(z),
                                                       z.stride(0), _p(out), out.stride(0), _dt(x), _stream()),
                   "hexmi_add_matmul_softmax")


_W8_WORKSPACES = {}          # (device index, stream) -> uint8 tensor, grown on demand


def _w8a16_impl(a, w, scales, out):
    M, K = a.shape
    N = w.shape[0]
    with _on(a.device):
        # shapes the library sums over several K parts need fp32 scratch for the partial tiles; one buffer per device
        # and stream is kept and reused (calls on one stream are ordered, so they may share it)
        need = (_lib.lib().hexmi_gemm_w8a16_workspace(M, N, K) if _lib.lib().hexmi_gemm_w8a16_workspace_helps(M, N, K)
                else 0)
        ws = None
        if need:
            key = (a.device.index, _stream())
            ws = _W8_WORKSPACES.get(key)
            if ws is None or ws.numel() < need:
                ws = torch.empty(need, dtype=torch.uint8, device=a.device)
                _W8_WORKSPACES[key] = ws
        _lib.check(_lib.lib().hexmi_gemm_w8a16_ws(M, N, K, _p(a), _p(w), _p(scales), _p(out), _p(ws),
                                                  ws.numel() if ws is not None else 0, _stream()),
                   "hexmi_gemm_w8a16_ws")


def _pack_impl(w, out):
    N, K = w.shape
    with _on(w.device):
        _lib.check(_lib.lib().hexmi_pack_w8(N, K, _p(w), _p(out), _stream()), "hexmi_pack_w8")


def _w8a16_packed_impl(a, wp, scales, out):
    M, K = a.shape
    N = scales.shape[0]
    with _on(a.device):
        _lib.check(_lib.lib().hexmi_gemm_w8a16_packed(M, N, K, _p(a), _p(wp), _p(scales), _p(out), _stream()),
                   "hexmi_gemm_w8a16_packed")


def _dequant_impl(w, scales, out):
    N, K = w.shape
    with _on(w.device):
        _lib.check(_lib.lib().hexmi_dequant_w8(N, K, _p(w), _p(scales), _p(out), _stream()), "hexmi_dequant_w8")


def _flash_impl(q, k, v, sm_scale, causal, out):
    Z, H, S, D = q.shape
    with _on(q.device):
        _lib.check(_lib.lib().hexmi_flash_attn_fwd(_p(q), _p(k), _p(v), _p(out), Z, H, S, D, sm_scale,
                                                   1 if causal else 0, _dt(q), _dt(out), _stream()),
                   "hexmi_flash_attn_fwd")


_Strides9 = ctypes.c_int64 * 9


def _flash_strided(q, k, v, sm_scale, causal, out):
    """Attention over device tensors read where they stand: True if the library takes their strides."""
    Z, H, S, D = q.shape
    strides = _Strides9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    with _on(q.device):
        status = _lib.lib().hexmi_flash_attn_fwd_strided(_p(q), _p(k), _p(v), _p(out), Z, H, S, D, strides, sm_scale,
                                                         1 if causal else 0, _dt(q), _dt(out), _stream())
    if status == _lib.ENOTSUP:
        return False
    _lib.check(status, "hexmi_flash_attn_fwd_strided")
    return True


def _attention_impl(q, k, v, mask, sm_scale, out):
    B, Sq, D = q.shape
    Skv = k.shape[1]
    with _on(q.device):
        # few queries over many keys: the keys are cut over several workgroups when the library is handed scratch for
        # their fp32 sums; the question costs 0.9 us and is not asked where the answer is always none
        need = (_lib.lib().hexmi_attention_workspace(B, Sq, Skv, D, 0 if mask is None else 1, _dt(q))
                if Skv > _lib.ATTENTION_ONE_LAUNCH_KEYS else 0)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _lib.check(_lib.lib().hexmi_attention_ws(_p(q), _p(k), _p(v), _p(mask), _p(out), B, Sq, Skv, D, sm_scale,
                                                 _dt(q), _dt(out), _p(ws), need, _stream()), "hexmi_attention_ws")


def _unary_impl(op, x, out):
    with _on(x.device):
        _lib.check(_lib.lib().hexmi_unary(op, _p(x), _p(out), x.numel(), _dt(x), _stream()), "hexmi_unary")


def _binary_impl(op, a, b, out):
    with _on(a.device):
        _lib.check(_lib.lib().hexmi_binary(op, _p(a), _p(b), _p(out), a.numel(), _dt(a), _stream()), "hexmi_binary")


def _block_sum_impl(x, block, out):
    n = x.numel()
    need = _lib.lib().hexmi_block_sum_workspace(n, block, _dt(x))
    # huge programs (the reference test sums 2^20 elements in one) are summed in two passes over the whole chip
    # when the library is handed scratch for its fp32 partial sums
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with _on(x.device):
        _lib.check(_lib.lib().hexmi_block_sum_ws(_p(x), _p(out), n, block, _dt(x), _p(ws), need, _stream()),
                   "hexmi_block_sum_ws")


def _rope_impl(x, theta, out):
    B, L, H, D = x.shape
    with _on(x.device):
        _lib.check(_lib.lib().hexmi_rope(_p(x), _p(out), B, L, H, D, theta, _dt(x), _stream()), "hexmi_rope")


_PAIRS = {"adjacent": 0, "halves": 1}


def _strides(t):
    """A tensor's strides; a dimension of one has none that matters."""
    return [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]


def _head_rows(x, out=None, weight=None):
    """hexmi_head_rows of x [tokens, heads, dim] (and of out, where its rows go)."""
    if x is None:
        return None
    xs, os = _strides(x), (0, 0) if out is None else _strides(out)
    return _lib.HeadRows(_p(x), _p(out), _p(weight), x.shape[1], xs[0], xs[1], os[0], os[1])


def _rotation(inv_freq, eps, pairs):
    return _lib.Rotation(_p(inv_freq), 0 if inv_freq is None else 2 * inv_freq.numel(), _PAIRS[pairs], eps)


def _paged_batch(tokens, k_pages, v_pages, page_table, lengths, starts):
    n, heads, size, dim = k_pages.shape
    ks, vs = _strides(k_pages), _strides(v_pages)
    return _lib.PagedBatch(_p(k_pages), _p(v_pages), *ks[:3], *vs[:3], n, size, heads, dim, _p(page_table), page_table.stride(0),
                           page_table.shape[1], _p(lengths), _p(starts), lengths.shape[0], tokens)


def _qk_norm_rope_impl(q, k, q_weight, k_weight, inv_freq, positions, eps, pairs, q_out, k_out):
    with _on(q.device):
        _lib.check(_lib.lib().hexmi_qk_norm_rope(_head_rows(q, q_out, q_weight), _head_rows(k, k_out, k_weight),
                                                 _rotation(inv_freq, eps, pairs), _p(positions),
                                                 1 if positions is not None and positions.dtype == torch.int64 else 0, q.shape[0],
                                                 q.shape[2], _dt(q), _stream()), "hexmi_qk_norm_rope")


def _paged_append_impl(k, v, k_pages, v_pages, page_table, lengths, starts, k_weight, inv_freq, eps, pairs, q, q_weight, q_out):
    with _on(k_pages.device):
        _lib.check(_lib.lib().hexmi_paged_append(_head_rows(k, None, k_weight), _head_rows(v), _head_rows(q, q_out, q_weight),
                                                 _rotation(inv_freq, eps, pairs),
                                                 _paged_batch(k.shape[0], k_pages, v_pages, page_table, lengths, starts), _dt(k),
                                                 _stream()), "hexmi_paged_append")


def _paged_attention_impl(q, k_pages, v_pages, page_table, lengths, starts, sm_scale, shared_pages, out):
    batch = _paged_batch(q.shape[0], k_pages, v_pages, page_table, lengths, starts)
    shared = 0 if shared_pages is None else shared_pages.shape[0]
    with _on(q.device):
        need = _lib.lib().hexmi_paged_attention_workspace(batch, q.shape[1], shared)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _lib.check(_lib.lib().hexmi_paged_attention(_head_rows(q, out), batch, _p(shared_pages), shared, sm_scale, _dt(q), _p(ws), need,
                                                    _stream()), "hexmi_paged_attention")


for _name, _fn in (("softmax", _softmax_impl), ("rms_norm", _rms_norm_impl), ("layer_norm", _layer_norm_impl),
                   ("matmul", _matmul_impl), ("linear", _linear_impl), ("add_matmul_softmax", _add_matmul_softmax_impl),
                   ("w8a16_matmul", _w8a16_impl), ("dequant_w8", _dequant_impl), ("pack_w8", _pack_impl),
                   ("w8a16_matmul_packed", _w8a16_packed_impl),
                   ("flash_attention", _flash_impl), ("attention", _attention_impl),
                   ("unary", _unary_impl), ("binary", _binary_impl), ("block_sum", _block_sum_impl),
                   ("rope", _rope_impl), ("qk_norm_rope", _qk_norm_rope_impl), ("paged_append", _paged_append_impl),
                   ("paged_attention", _paged_attention_impl)):
    _LIBDEF.impl(_name, _fn, "CUDA")


# --------------------------------------------------------------------------
# staging helpers
# --------------------------------------------------------------------------
def _device():
    if not torch.cuda.is_available():
        raise RuntimeError("hexmi needs a GPU (gfx950); there is no CPU path")
    _lib.lib()
    return torch.device("cuda", torch.cuda.current_device())


def _stage(t, dev):
    """Contiguous device copy (or the tensor itself when it already is one)."""
    if t is None:
        return None
    if t.device.type != "cuda":
        t = t.to(dev, non_blocking=False)
    return t if t.is_contiguous() else t.contiguous()


def _span(t):
    """The addresses from a tensor's first element to behind its last."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlaps(t, *others):
    """Whether t may share memory with any of others, of one storage or not (an import over DLPack has a storage of its own)."""
    lo, hi = _span(t)
    return any(a < hi and lo < b for a, b in map(_span, others))


def _finish(result, out):
    """Write `result` (device) into the caller's `out` if they are different tensors."""
    if out is None:
        return result
    if out.data_ptr() != result.data_ptr() or out.device != result.device:
        out.copy_(result)
    return out


def _out_like(out, shape, dtype, dev):
    """Device tensor to compute into: `out` itself when usable, else a fresh one."""
    if out is not None:
        if tuple(out.shape) != tuple(shape):
            raise ValueError("hexmi: out has shape %s, expected %s" % (tuple(out.shape), tuple(shape)))
        if out.dtype != dtype:
            raise TypeError("hexmi: out has dtype %s, expected %s" % (out.dtype, dtype))
        if out.device.type == "cuda" and out.is_contiguous():
            return out
    return torch.empty(shape, dtype=dtype, device=dev)


# --------------------------------------------------------------------------
# public operators. A call of the usual form goes through csrc/torch_front.cpp, whose time is little more than its launch (4.9 us
# against 11.9 for a layer norm of 512 x 768). Any other calls the implementations above directly: the same code
# `torch.ops.hexmi.*` runs, without the dispatcher's round trip into Python (several microseconds).
# A caller that traces a model (torch.compile, FakeTensor propagation) needs the operators to appear as
# `torch.ops.hexmi.*` nodes: `through_dispatcher(True)` routes the operators that have a registered schema through
# the dispatcher (2-D operands, no column blocks; anything else keeps the direct call).
# --------------------------------------------------------------------------
_THROUGH_DISPATCHER = False


def through_dispatcher(enable=True):
    """Route softmax / rms_norm / layer_norm / matmul / w8a16_matmul / flash_attention through `torch.ops.hexmi.*`
    (visible to tracing) instead of calling the library directly. Returns the previous setting."""
    global _THROUGH_DISPATCHER
    previous, _THROUGH_DISPATCHER = _THROUGH_DISPATCHER, bool(enable)
    return previous


class _Front:
    """hexmi._front (csrc/torch_front.cpp), imported at the first call: a function of it takes a call of the plain form (dense
    device tensors, nothing optional but operands) and returns its result, or None for any other call. Where it is not built or
    was built for another torch or Python, a warning, and every call goes through ctypes."""

    def __getattr__(self, name):
        _lib.lib()
        names = ("softmax", "rms_norm", "layer_norm", "matmul", "w8a16_matmul", "flash_attention", "attention", "unary", "binary",
                 "qk_norm_rope", "paged_append", "paged_attention")
        if name not in names:
            raise AttributeError(name)
        try:
            from . import _front as native
            if native.torch_version != torch.__version__:
                raise ImportError("built for torch %s, not %s" % (native.torch_version, torch.__version__))
        except ImportError as e:
            warnings.warn("hexmi/_front.so is missing or does not load (%s): every call takes the slower route through ctypes; "
                          "build it with `python hexagon-mlir_amd/build.py`" % e, RuntimeWarning, stacklevel=3)
            native = None
        else:
            native.set_check(_lib.check)
        for f in names:
            setattr(self, f, getattr(native, f) if native else _not_plain)
        return getattr(self, name)


def _not_plain(*args):
    return None


_front = _Front()


def _run(name, impl, simple, *args):
    """impl(*args) directly, or torch.ops.hexmi.<name>(*simple) when tracing asked for the dispatcher and the call
    has the registered operator's form (simple is not None)."""
    if _THROUGH_DISPATCHER and simple is not None:
        getattr(torch.ops.hexmi, name)(*simple)
    else:
        impl(*args)


def _row_strided(t):
    """A 2-D device tensor whose rows are contiguous but not adjacent (a column slice, a padded buffer): the row
    operators read and write it in place through its row stride, as the reference's kernels take a memref with
    strides (test/utils/dsp/include/common.h:15-21)."""
    return (t is not None and t.device.type == "cuda" and t.dim() == 2 and t.stride(1) == 1
            and t.stride(0) >= t.shape[1] and not t.is_contiguous())


def _row_operands(x, out, dev):
    """(x on the device, tensor to compute into, rows, cols) with rows / cols None when both are 2-D strided views."""
    cols = x.shape[-1]
    rows = x.numel() // max(cols, 1)
    if _row_strided(x) or (_row_strided(out) and x.dim() == 2):
        xd = x if x.device.type == "cuda" and x.dim() == 2 and x.stride(1) == 1 else _stage(x, dev)
        if out is not None and (tuple(out.shape) != tuple(x.shape) or out.dtype != x.dtype):
            raise ValueError("hexmi: out must have the shape and dtype of x")
        od = out if (out is not None and out.device.type == "cuda" and out.stride(1) == 1) else torch.empty_like(xd, memory_format=torch.contiguous_format)
        return xd, od, None, None
    return _stage(x, dev), _out_like(out, x.shape, x.dtype, dev), rows, cols


def softmax(x, out=None, dim=-1, block_cols=0):
    """Softmax over the last dimension (`F.softmax(x, dim=1)` of
    test/python/triton/test_softmax.py:93 for 2-D input). block_cols > 0: the two-phase (online) form of
    test/python/triton/test_online_softmax.py:31-81 over column blocks of that size."""
    if out is None and dim == -1 and not block_cols and not _THROUGH_DISPATCHER:
        y = _front.softmax(x)
        if y is not None:
            return y
    if dim not in (-1, x.dim() - 1):
        raise ValueError("hexmi.softmax reduces over the last dimension only")
    if x.dim() < 1:
        raise ValueError("hexmi.softmax needs at least 1 dimension")
    dev = _device() if x.device.type != "cuda" else x.device
    xd, od, rows, cols = _row_operands(x, out, dev)
    _run("softmax", _softmax_impl, (xd, od) if xd.dim() == 2 and not block_cols else None, xd, od, rows, cols, int(block_cols))
    return _finish(od, out)


def rms_norm(x, weight=None, eps=1e-5, out=None, block_cols=0):
    """`F.rms_norm(x, (C,), weight, eps)` (test/python/triton/test_rms_norm.py:85-87)."""
    if out is None and not block_cols and not _THROUGH_DISPATCHER:
        y = _front.rms_norm(x, weight, eps)
        if y is not None:
            return y
    dev = _device() if x.device.type != "cuda" else x.device
    cols = x.shape[-1]
    if weight is not None and (weight.shape != (cols,) or weight.dtype != x.dtype):
        raise ValueError("hexmi.rms_norm: weight must be [%d] of %s" % (cols, x.dtype))
    xd, od, rows, c = _row_operands(x, out, dev)
    wd = _stage(weight, dev)
    _run("rms_norm", _rms_norm_impl, (xd, wd, float(eps), od) if xd.dim() == 2 and not block_cols else None,
         xd, wd, float(eps), od, rows, c, int(block_cols))
    return _finish(od, out)


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None, mean=None, rstd=None, block_cols=0):
    """`F.layer_norm(x, (C,), weight, bias, eps)` (test/python/triton/test_layer_norm.py:111-113);
    `mean` / `rstd` (fp32, one per row) are filled when given, as the reference kernel does."""
    if out is None and mean is None and rstd is None and not block_cols and not _THROUGH_DISPATCHER:
        y = _front.layer_norm(x, weight, bias, eps)
        if y is not None:
            return y
    dev = _device() if x.device.type != "cuda" else x.device
    cols = x.shape[-1]
    nrows = x.numel() // max(cols, 1)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (cols,) or t.dtype != x.dtype):
            raise ValueError("hexmi.layer_norm: %s must be [%d] of %s" % (name, cols, x.dtype))
    xd, od, rows, c = _row_operands(x, out, dev)
    wd, bd = _stage(weight, dev), _stage(bias, dev)
    md = None if mean is None else _out_like(mean if mean.dtype == torch.float32 else None, (nrows,), torch.float32, dev)
    rd = None if rstd is None else _out_like(rstd if rstd.dtype == torch.float32 else None, (nrows,), torch.float32, dev)
    _run("layer_norm", _layer_norm_impl, (xd, wd, bd, float(eps), od, md, rd) if xd.dim() == 2 and not block_cols else None,
         xd, wd, bd, float(eps), od, md, rd, rows, c, int(block_cols))
    if mean is not None:
        _finish(md, mean)
    if rstd is not None:
        _finish(rd, rstd)
    return _finish(od, out)


def matmul(a, b, out=None, out_dtype=None, trans_b=False, bias=None, residual=None):
    """C = A @ B (or A @ B.T when trans_b), fp16/bf16 inputs with fp32 accumulation on the matrix cores, or fp32
    inputs multiplied in fp32. out_dtype: the input dtype (default) or torch.float32
    (test/python/triton/test_matmul.py:35-91; docs/tutorials/triton/matmul_hexkl.md:61-111).
    bias [N] and residual [M,N] (of the output dtype) are added to the fp32 sums inside the GEMM kernel, the way the
    reference's fusion pass pulls the consumers of a matmul into its loop nest
    (qcom_hexagon_backend/lib/Conversion/LinalgToLLVM/LinalgToLLVMPass.cpp:280-283): C = A @ B + bias + residual
    with one rounding and no extra launch."""
    if out is None and out_dtype is None and not _THROUGH_DISPATCHER:
        y = _front.matmul(a, b, trans_b, bias, residual)
        if y is not None:
            return y
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("hexmi.matmul takes 2-D tensors")
    if a.dtype != b.dtype or a.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("hexmi.matmul: A and B must both be float16, both bfloat16 or both float32")
    if a.dtype == torch.float32 and (out_dtype or (out.dtype if out is not None else torch.float32)) != torch.float32:
        raise TypeError("hexmi.matmul: float32 operands give a float32 result")
    M, K = a.shape
    N = b.shape[0] if trans_b else b.shape[1]
    if (b.shape[1] if trans_b else b.shape[0]) != K:
        raise ValueError("hexmi.matmul: inner dimensions differ: %s x %s" % (tuple(a.shape), tuple(b.shape)))
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else a.dtype
    if bias is not None and (bias.shape != (N,) or bias.dtype != out_dtype):
        raise ValueError("hexmi.matmul: bias must be [N] of the output dtype")
    if residual is not None and (residual.shape != (M, N) or residual.dtype != out_dtype):
        raise ValueError("hexmi.matmul: residual must be [M,N] of the output dtype")
    dev = _device() if a.device.type != "cuda" else a.device
    ad, bd = _stage(a, dev), _stage(b, dev)
    od = _out_like(out, (M, N), out_dtype, dev)
    if bias is None and residual is None:
        _run("matmul", _matmul_impl, (ad, bd, bool(trans_b), od), ad, bd, bool(trans_b), od)
    else:
        _linear_impl(ad, bd, _stage(bias, dev), _stage(residual, dev), bool(trans_b), od)
    return _finish(od, out)


def pack_weight(w):
    """One-time re-layout of a constant 16-bit weight [K,N] into the K-contiguous form [N,K] the GEMM streams fastest;
    multiply with `matmul(a, packed, trans_b=True)`. The analogue of the reference folding the transpose of a
    constant weight at compile time (qcom_hexagon_backend/lib/Transforms/FoldResourceTransposePass.cpp:21-110)."""
    if w.dim() != 2 or w.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("hexmi.pack_weight: expected a 2-D float16 or bfloat16 tensor")
    dev = _device() if w.device.type != "cuda" else w.device
    wd = _stage(w, dev)
    rows, cols = wd.shape
    out = torch.empty((cols, rows), dtype=w.dtype, device=dev)
    with _on(dev):
        _lib.check(_lib.lib().hexmi_transpose16(rows, cols, _p(wd), wd.stride(0), _p(out), out.stride(0), _stream()),
                   "hexmi_transpose16")
    return out


def _quant_params(name, w_int8, scales, zero_points):
    """Checks the parameters of `f = (float(q) - zero_point) * scale`; returns per_tensor (one scale, and one zero
    point, for the whole tensor) against per output channel."""
    if w_int8.dtype != torch.int8 or scales.dtype != torch.float16:
        raise TypeError("hexmi.%s: expected int8 weights, fp16 scales" % name)
    if w_int8.dim() != 2 or scales.dim() != 1 or scales.shape[0] not in (1, w_int8.shape[0]):
        raise ValueError("hexmi.%s: shapes W[N,K] and scales[N] (per channel) or scales[1] (per tensor) required" % name)
    per_tensor = scales.shape[0] == 1 and w_int8.shape[0] != 1
    if zero_points is not None:
        if zero_points.dtype != torch.int8:
            raise TypeError("hexmi.%s: zero points are int8" % name)
        if zero_points.shape != scales.shape:
            raise ValueError("hexmi.%s: zero_points must have the shape of scales" % name)
    return per_tensor


def w8a16_matmul(a, w_int8, scales, out=None, zero_points=None):
    """C[m,n] = sum_k A[m,k] * ((W[n,k] - zero_points[n]) * scales[n]); A fp16 [M,K], W int8 [N,K], scales fp16 [N]
    (or [1]: one scale and zero point for the tensor), zero_points int8 or None (symmetric)."""
    if out is None and not _THROUGH_DISPATCHER:
        y = _front.w8a16_matmul(a, w_int8, scales, zero_points)
        if y is not None:
            return y
    if a.dtype != torch.float16:
        raise TypeError("hexmi.w8a16_matmul: expected fp16 activations, int8 weights, fp16 scales")
    if w_int8.dtype != torch.int8 or scales.dtype != torch.float16:
        raise TypeError("hexmi.w8a16_matmul: expected fp16 activations, int8 weights, fp16 scales")
    if a.dim() != 2 or w_int8.dim() != 2 or a.shape[1] != w_int8.shape[1]:
        raise ValueError("hexmi.w8a16_matmul: shapes A[M,K], W[N,K], scales[N] required")
    per_tensor = _quant_params("w8a16_matmul", w_int8, scales, zero_points)
    dev = _device() if a.device.type != "cuda" else a.device
    ad, wd, sd = _stage(a, dev), _stage(w_int8, dev), _stage(scales, dev)
    od = _out_like(out, (a.shape[0], w_int8.shape[0]), torch.float16, dev)
    if zero_points is None and not per_tensor:
        _run("w8a16_matmul", _w8a16_impl, (ad, wd, sd, od), ad, wd, sd, od)
    else:
        zd = _stage(zero_points, dev)
        M, K = ad.shape
        with _on(ad.device):
            _lib.check(_lib.lib().hexmi_gemm_w8a16_ex(M, wd.shape[0], K, _p(ad), _p(wd), _p(sd), _p(zd),
                                                      1 if per_tensor else 0, _p(od), _stream()), "hexmi_gemm_w8a16_ex")
    return _finish(od, out)


def pack_w8(w_int8):
    """One-time re-layout of int8 weights [N,K] (K % 64 == 0) into the fragment-major order `w8a16_matmul_packed`
    reads (flat int8 tensor of ceil(N/16)*16*K bytes); the analogue of the reference's constant-weight
    pre-processing (qcom_hexagon_backend/lib/Transforms/PreprocessWeightsForHMXPass.cpp:39-117)."""
    if w_int8.dtype != torch.int8 or w_int8.dim() != 2:
        raise TypeError("hexmi.pack_w8: expected an int8 [N,K] tensor")
    N, K = w_int8.shape
    if K % 64 != 0:
        raise ValueError("hexmi.pack_w8: K must be a multiple of 64")
    dev = _device() if w_int8.device.type != "cuda" else w_int8.device
    wd = _stage(w_int8, dev)
    out = torch.empty(((N + 15) // 16) * 16 * K, dtype=torch.int8, device=dev)
    _pack_impl(wd, out)
    return out


def w8a16_matmul_packed(a, w_packed, scales, out=None):
    """`w8a16_matmul` on weights packed by `pack_w8` (N = len(scales)). `w8a16_matmul` uses kernels that
    sum in another order (one fp16 ulp)."""
    if a.dtype != torch.float16 or w_packed.dtype != torch.int8 or scales.dtype != torch.float16:
        raise TypeError("hexmi.w8a16_matmul_packed: expected fp16 activations, packed int8 weights, fp16 scales")
    if a.dim() != 2 or scales.dim() != 1:
        raise ValueError("hexmi.w8a16_matmul_packed: shapes A[M,K], scales[N] required")
    M, K = a.shape
    N = scales.shape[0]
    if w_packed.numel() != ((N + 15) // 16) * 16 * K:
        raise ValueError("hexmi.w8a16_matmul_packed: packed weights do not match N=%d, K=%d" % (N, K))
    dev = _device() if a.device.type != "cuda" else a.device
    ad, wd, sd = _stage(a, dev), _stage(w_packed, dev), _stage(scales, dev)
    od = _out_like(out, (M, N), torch.float16, dev)
    _w8a16_packed_impl(ad, wd, sd, od)
    return _finish(od, out)


def dequant_w8(w_int8, scales, out=None, zero_points=None):
    """fp32 [N,K] = (float(W[n,k]) - zero_points[n]) * float(scales[n]) (the dequantisation the fused kernel applies;
    scales / zero_points of one element: per tensor)."""
    per_tensor = _quant_params("dequant_w8", w_int8, scales, zero_points)
    dev = _device() if w_int8.device.type != "cuda" else w_int8.device
    wd, sd = _stage(w_int8, dev), _stage(scales, dev)
    od = _out_like(out, w_int8.shape, torch.float32, dev)
    if zero_points is None and not per_tensor:
        _dequant_impl(wd, sd, od)
    else:
        zd = _stage(zero_points, dev)
        with _on(wd.device):
            _lib.check(_lib.lib().hexmi_dequant_w8_ex(wd.shape[0], wd.shape[1], _p(wd), _p(sd), _p(zd),
                                                      1 if per_tensor else 0, _p(od), _stream()), "hexmi_dequant_w8_ex")
    return _finish(od, out)


def flash_attention(q, k, v, sm_scale=None, causal=False, out=None, out_dtype=None):
    """softmax(sm_scale * Q K^T [+causal]) V for [Z,H,S,D] tensors
    (`F.scaled_dot_product_attention(q, k, v, scale=...)`, test/python/triton/test_flash_attention.py:212)."""
    if out is None and out_dtype is None and not _THROUGH_DISPATCHER:
        y = _front.flash_attention(q, k, v, sm_scale, causal)
        if y is not None:
            return y
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("hexmi.flash_attention: q, k, v must share one [Z,H,S,D] shape")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("hexmi.flash_attention: q, k, v dtypes differ")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else q.dtype
    dev = _device() if q.device.type != "cuda" else q.device
    od = _out_like(out, q.shape, out_dtype, dev)
    # slices of one projection and transposed heads are read where they stand (three copies, 5 us each for 2 x 12 x 1000 x 64)
    if (not _THROUGH_DISPATCHER and (out is None or not _overlaps(od, q, k, v))
            and not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous())
            and q.device == k.device == v.device == od.device
            and q.stride(3) == k.stride(3) == v.stride(3) == 1
            and _flash_strided(q, k, v, float(sm_scale), causal, od)):
        return _finish(od, out)
    qd, kd, vd = _stage(q, dev), _stage(k, dev), _stage(v, dev)
    _run("flash_attention", _flash_impl, (qd, kd, vd, float(sm_scale), bool(causal), od), qd, kd, vd, float(sm_scale), bool(causal), od)
    return _finish(od, out)


def attention(q, k, v, mask=None, sm_scale=None, out=None, out_dtype=None):
    """tm_tensor.attention: softmax(Q K^T / sqrt(d) + mask) V for q [B,Sq,D], k / v [B,Skv,D] and an additive
    mask [B,Sq,Skv] (or None) (include/hexagon/Dialect/TmTensor/IR/TmTensorOps.td:28-56,
    lib/Transforms/LowerTmTensor.cpp:70-235); `F.scaled_dot_product_attention(q, k, v, attn_mask=mask)`."""
    if out is None and out_dtype is None:
        y = _front.attention(q, k, v, mask, sm_scale)
        if y is not None:
            return y
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("hexmi.attention: q [B,Sq,D], k and v [B,Skv,D]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("hexmi.attention: q, k, v dtypes differ")
    B, Sq, D = q.shape
    Skv = k.shape[1]
    if mask is not None and (tuple(mask.shape) != (B, Sq, Skv) or mask.dtype != q.dtype):
        raise ValueError("hexmi.attention: mask must be [%d,%d,%d] of %s" % (B, Sq, Skv, q.dtype))
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else q.dtype
    dev = _device() if q.device.type != "cuda" else q.device
    qd, kd, vd, md = _stage(q, dev), _stage(k, dev), _stage(v, dev), _stage(mask, dev)
    od = _out_like(out, q.shape, out_dtype, dev)
    _attention_impl(qd, kd, vd, md, float(sm_scale), od)
    return _finish(od, out)


UNARY_OPS = {"gelu_tanh": 0, "silu": 1, "rsqrt": 2, "sin": 3, "cos": 4, "exp": 5}
BINARY_OPS = {"add": 0, "sub": 1, "mul": 2, "div": 3}


def unary(op, x, out=None):
    """Element-wise `op` in UNARY_OPS ("gelu_tanh": test/python/triton/test_gelu.py:43-54, "silu": test_silu.py:43-52,
    "rsqrt": test_rsqrt.py:20-24, "sin" / "cos": test_math_ops.py:25-38, "exp")."""
    if op not in UNARY_OPS:
        raise ValueError("hexmi.unary: unknown op %r" % (op,))
    if out is None:
        y = _front.unary(UNARY_OPS[op], x)
        if y is not None:
            return y
    dev = _device() if x.device.type != "cuda" else x.device
    xd = _stage(x, dev)
    od = _out_like(out, x.shape, x.dtype, dev)
    _unary_impl(UNARY_OPS[op], xd, od)
    return _finish(od, out)


def gelu(x, out=None):
    """`F.gelu(x, approximate="tanh")` (test/python/triton/test_gelu.py:73)."""
    return unary("gelu_tanh", x, out)


def silu(x, out=None):
    """`F.silu(x)` (test/python/triton/test_silu.py:69)."""
    return unary("silu", x, out)


def binary(op, a, b, out=None):
    """Element-wise a (op) b for same-shape tensors, op in BINARY_OPS (test/python/triton/test_vec_add.py,
    test_vec_div_2d.py:21-55)."""
    if op not in BINARY_OPS:
        raise ValueError("hexmi.binary: unknown op %r" % (op,))
    if out is None:
        y = _front.binary(BINARY_OPS[op], a, b)
        if y is not None:
            return y
    if a.shape != b.shape or a.dtype != b.dtype:
        raise ValueError("hexmi.binary: operands must share shape and dtype")
    dev = _device() if a.device.type != "cuda" else a.device
    ad, bd = _stage(a, dev), _stage(b, dev)
    od = _out_like(out, a.shape, a.dtype, dev)
    _binary_impl(BINARY_OPS[op], ad, bd, od)
    return _finish(od, out)


def block_sum(x, block=None, out=None):
    """out[p] = sum of the p-th run of `block` elements of x (flattened); block=None sums everything into out[0]
    (`torch.sum(x)`, test/python/triton/test_sum.py:30-47)."""
    n = x.numel()
    if block is None:
        block = max(n, 1)
    if block < 1:
        raise ValueError("hexmi.block_sum: block must be positive")
    programs = (n + block - 1) // block
    dev = _device() if x.device.type != "cuda" else x.device
    xd = _stage(x, dev).reshape(-1)
    od = _out_like(out, (programs,), x.dtype, dev)
    _block_sum_impl(xd, int(block), od)
    return _finish(od, out)


def rope(x, theta=10000.0, out=None):
    """Rotary embedding of x [batch, seq, heads, features] over adjacent feature pairs
    (`rope_reference_pytorch`, test/python/triton/test_rope.py:60-95)."""
    if x.dim() != 4 or x.shape[-1] % 2 != 0:
        raise ValueError("hexmi.rope: x must be [batch, seq, heads, features] with an even feature count")
    dev = _device() if x.device.type != "cuda" else x.device
    xd = _stage(x, dev)
    od = _out_like(out, x.shape, x.dtype, dev)
    _rope_impl(xd, float(theta), od)
    return _finish(od, out)


def rope_frequencies(columns, theta=10000.0, device=None):
    """The angles per position, theta^(-2i / columns), of a rotation of `columns` columns of a head, as the float64 tensor that
    `qk_norm_rope` and `paged_append` take (`compute_thetas`, test/python/triton/test_rope.py:43-57): made once by a program, on the
    GPU, and scaled there for contexts longer than a model's own."""
    if columns < 2 or columns % 2 != 0:
        raise ValueError("hexmi.rope_frequencies: columns must be even and positive")
    if not theta > 0:
        raise ValueError("hexmi.rope_frequencies: theta must be positive")
    i = torch.arange(0, columns, 2, dtype=torch.float64)
    return (float(theta) ** (-i / columns)).to(_device() if device is None else device)


def _rows_of_heads(t, dev):
    """t [tokens, heads, dim] on the device, its columns adjacent: slices of one projection are read where they stand."""
    if t is None:
        return None
    if t.device.type != "cuda":
        t = t.to(dev, non_blocking=False)
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _apart(a, b):
    """Whether two tensors share no memory: their spans lie apart, or they are column slices of the same rows."""
    if not _overlaps(a, b):
        return True
    pitch = a.stride(0)
    if pitch != b.stride(0) or a.element_size() != b.element_size() or (a.data_ptr() - b.data_ptr()) % a.element_size():
        return False
    wide = [sum((n - 1) * s for n, s in zip(t.shape[1:], t.stride()[1:])) + 1 for t in (a, b)]
    ahead = (a.data_ptr() - b.data_ptr()) // a.element_size() % pitch if pitch else 0
    return ahead >= wide[1] and ahead + wide[0] <= pitch


def _rows_out(name, out, x, others, dev):
    """Where rows like x's are computed: out where it is a device tensor that shares no memory with what is read (but for x itself, row
    for row), or fresh memory."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=dev)
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("hexmi.%s: out must be %s of %s" % (name, tuple(x.shape), x.dtype))
    own = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    plain = out.device == dev and (out.stride(2) == 1 or out.shape[2] == 1) and all(s > 0 or n == 1 for n, s in zip(out.shape, out.stride()))
    if plain and out.numel() and (own or _apart(out, x)) and all(_apart(out, t) for t in others if t is not None and t.numel()):
        return out
    return torch.empty(x.shape, dtype=x.dtype, device=dev)


def _head_operands(name, x, weight, dim, dtype):
    if x.dim() != 3 or x.shape[1] < 1 or x.shape[2] != dim or dim < 1:
        raise ValueError("hexmi.%s: rows of heads are [tokens, heads, %s]" % (name, dim))
    if x.dtype != dtype:
        raise TypeError("hexmi.%s: operands must share one type" % name)
    if weight is not None and (weight.shape != (dim,) or weight.dtype != dtype):
        raise ValueError("hexmi.%s: a weight must be [%d] of %s" % (name, dim, dtype))


def _check_rotation(name, inv_freq, pairs, dim):
    if pairs not in _PAIRS:
        raise ValueError("hexmi.%s: pairs are 'adjacent' or 'halves'" % name)
    if inv_freq is not None:
        if inv_freq.dtype != torch.float64:
            raise TypeError("hexmi.%s: inv_freq is float64 (hexmi.rope_frequencies makes it)" % name)
        if inv_freq.dim() != 1 or 2 * inv_freq.numel() > dim:
            raise ValueError("hexmi.%s: inv_freq is [rotated columns / 2], at most %d" % (name, dim // 2))


def _one_device(name, dev, *tensors):
    for t in tensors:
        if t is not None and t.device.type == "cuda" and t.device != dev:
            raise ValueError("hexmi.%s: operands are on %s and %s" % (name, dev, t.device))


def qk_norm_rope(q, k=None, q_weight=None, k_weight=None, inv_freq=None, positions=None, eps=1e-5, pairs="adjacent", q_out=None,
                 k_out=None):
    """RMS norm of every head's row of q [tokens, heads, dim] and k [tokens, kv heads, dim] (each where it has a weight [dim]) and their
    rotation by the tokens' positions, in one pass and with one rounding: `rms_norm` and `rope` (test/python/triton/test_rms_norm.py:37-63,
    test_rope.py:97-197) at any positions.

    inv_freq (float64, `rope_frequencies`) turns 2 * len(inv_freq) leading columns, in pairs of columns (2i, 2i + 1) ("adjacent") or
    (i, i + len(inv_freq)) ("halves"); None: no rotation. positions: int32 or int64 [tokens]. q and k may be slices of one projection;
    q_out and k_out may be q and k. Returns q's rows, or with k the pair."""
    if q_out is None and k_out is None and not _THROUGH_DISPATCHER:
        y = _front.qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions, eps, pairs)
        if y is not None:
            return y
    name = "qk_norm_rope"
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("hexmi.qk_norm_rope: float16, bfloat16 or float32")
    dim = q.shape[-1]
    _head_operands(name, q, q_weight, dim, q.dtype)
    _check_rotation(name, inv_freq, pairs, dim)
    if k is not None:
        _head_operands(name, k, k_weight, dim, q.dtype)
        if k.shape[0] != q.shape[0]:
            raise ValueError("hexmi.qk_norm_rope: q and k have %d and %d tokens" % (q.shape[0], k.shape[0]))
    elif k_weight is not None or k_out is not None:
        raise ValueError("hexmi.qk_norm_rope: k_weight and k_out go with k")
    if inv_freq is not None and positions is None:
        raise ValueError("hexmi.qk_norm_rope: a rotation needs positions")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or positions.shape != (q.shape[0],)):
        raise ValueError("hexmi.qk_norm_rope: positions must be int32 or int64 [%d]" % q.shape[0])
    dev = _device() if q.device.type != "cuda" else q.device
    _one_device(name, dev, k, q_weight, k_weight, inv_freq, positions)
    qd, kd = _rows_of_heads(q, dev), _rows_of_heads(k, dev)
    qw, kw, fd, pd = _stage(q_weight, dev), _stage(k_weight, dev), _stage(inv_freq, dev), _stage(positions, dev)
    qo = _rows_out(name, q_out, qd, (kd, qw, kw, fd, pd), dev)
    ko = None if k is None else _rows_out(name, k_out, kd, (qd, qw, kw, fd, pd), dev)
    if ko is not None and qo.numel() and not _apart(qo, ko):
        raise ValueError("hexmi.qk_norm_rope: q_out and k_out share memory")
    if q.shape[0]:
        args = (qd, kd, qw, kw, fd, pd, float(eps), pairs, qo, ko)
        _run(name, _qk_norm_rope_impl, args, *args)
    q_done = _finish(qo, q_out)
    return q_done if k is None else (q_done, _finish(ko, k_out))


def _paged_operands(name, tokens, k_pages, v_pages, page_table, lengths, starts):
    """Checks a paged cache and its batch and returns (page_table, lengths, starts) on its device."""
    if k_pages.device.type != "cuda" or v_pages.device != k_pages.device:
        raise ValueError("hexmi.%s: the pages stay on the GPU" % name)
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.numel() == 0:
        raise ValueError("hexmi.%s: k_pages and v_pages are [pages, kv heads, page size, dim]" % name)
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("hexmi.%s: a key's columns must be adjacent" % name)
    for what, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1), ("starts", starts, 1)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != dims):
            raise ValueError("hexmi.%s: %s must be an int32 tensor of %d dimension%s" % (name, what, dims, "s" if dims > 1 else ""))
    n = lengths.shape[0]
    if page_table.shape[0] != n:
        raise ValueError("hexmi.%s: page_table has a row and lengths a value for each sequence" % name)
    if starts is None and n != tokens:
        raise ValueError("hexmi.%s: without starts every sequence has one new token (%d sequences, %d tokens)" % (name, n, tokens))
    if starts is not None and starts.shape[0] != n + 1:
        raise ValueError("hexmi.%s: starts must be [%d]" % (name, n + 1))
    dev = k_pages.device
    _one_device(name, dev, page_table, lengths, starts)
    table = page_table.to(dev)
    if table.numel() and (table.stride(1) != 1 and table.shape[1] > 1 or table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        table = table.contiguous()
    return table, _stage(lengths, dev), _stage(starts, dev)


def paged_append(k, v, k_pages, v_pages, page_table, lengths, starts=None, k_weight=None, inv_freq=None, eps=1e-5, pairs="adjacent",
                 q=None, q_weight=None, q_out=None):
    """Puts the keys and values of new tokens, [tokens, kv heads, dim], into the pages of their sequences, the keys normed (with k_weight)
    and rotated (with inv_freq) by their positions on the way, as `qk_norm_rope` does; with q [tokens, heads, dim], its rows too, which
    are returned.

    k_pages, v_pages [pages, kv heads, page size, dim] are changed in place (any strides: a cache that keeps the heads of a token side by
    side is a transposed view). page_table int32 [sequences, columns]: the pages of each sequence; an entry that is no page's number (-1,
    say) is none, and a token there is left out. lengths int32 [sequences]: the positions of each sequence, the new tokens included, which
    are its last. starts int32 [sequences + 1]: sequence b's tokens are the rows starts[b] .. starts[b + 1] - 1 (of those
    that there are); rows of no sequence (padding behind the last) leave nothing, and zeros in q's result. None: one token a sequence. What the index tensors hold is
    read on the GPU only, so the call can be captured into a graph and replayed as they change."""
    if q_out is None and not _THROUGH_DISPATCHER:
        y = _front.paged_append(k, v, k_pages, v_pages, page_table, lengths, starts, k_weight, inv_freq, eps, pairs, q, q_weight)
        if y is not None:
            return y if q is not None else None
    name = "paged_append"
    if k.dtype not in (torch.float16, torch.bfloat16) or k_pages.dtype != k.dtype:
        raise TypeError("hexmi.paged_append: keys and pages must both be float16 or both bfloat16")
    if k_pages.dim() != 4 or k.dim() != 3 or k.shape[1:] != (k_pages.shape[1], k_pages.shape[3]) or v.shape != k.shape:
        raise ValueError("hexmi.paged_append: k and v are [tokens, kv heads, dim], the pages [pages, kv heads, page size, dim]")
    dim, tokens = k.shape[2], k.shape[0]
    _head_operands(name, k, k_weight, dim, k.dtype)
    _head_operands(name, v, None, dim, k.dtype)
    _check_rotation(name, inv_freq, pairs, dim)
    if q is not None:
        _head_operands(name, q, q_weight, dim, k.dtype)
        if q.shape[0] != tokens:
            raise ValueError("hexmi.paged_append: q and k have %d and %d tokens" % (q.shape[0], tokens))
    elif q_weight is not None or q_out is not None:
        raise ValueError("hexmi.paged_append: q_weight and q_out go with q")
    table, lens, begin = _paged_operands(name, tokens, k_pages, v_pages, page_table, lengths, starts)
    dev = k_pages.device
    _one_device(name, dev, k, v, q, k_weight, q_weight, inv_freq)
    if k_pages.data_ptr() == v_pages.data_ptr():
        raise ValueError("hexmi.paged_append: keys and values need pages of their own")
    # rows that stand in the pages themselves (one sequence's going to another) are read before any is written
    kd, vd, qd = (t.clone() if t is not None and t.numel() and _overlaps(t, k_pages, v_pages) else t
                  for t in (_rows_of_heads(k, dev), _rows_of_heads(v, dev), _rows_of_heads(q, dev)))
    kw, qw, fd = _stage(k_weight, dev), _stage(q_weight, dev), _stage(inv_freq, dev)
    qo = None if q is None else _rows_out(name, q_out, qd, (kd, vd, kw, qw, fd, table, lens, begin, k_pages, v_pages), dev)
    if tokens:
        args = (kd, vd, k_pages, v_pages, table, lens, begin, kw, fd, float(eps), pairs, qd, qw, qo)
        _run(name, _paged_append_impl, args, *args)
    return None if q is None else _finish(qo, q_out)


def paged_attention(q, k_pages, v_pages, page_table, lengths, starts=None, sm_scale=None, shared_pages=None, out=None):
    """Attention of new tokens q [tokens, heads, dim] over a paged cache: row (t, h) is softmax(sm_scale * Q K^T) V over the keys of
    kv head h // (heads // kv heads) at the positions of its sequence up to its own (`attention` with a cache and masks of its own;
    test/python/triton/test_flash_attention.py:37-168). The cache and the batch are `paged_append`'s, which comes first: lengths counts
    the new tokens. One token a sequence (starts None) is a decode step, runs of tokens are prompts or pieces of them, and a batch may
    hold both.

    shared_pages int32 [n]: the first n pages of every sequence are these (a prompt that all have in common), and their keys are gone
    through once for all of them; the result is the same without, if the table names them.

    How the work is cut goes by the width of page_table: one much wider than the longest sequence costs a small batch 2 to 10 us, and sums in
    another order.

    A row without any key, and a row of no sequence, is zeros. What the pages hold past a sequence's length is not used, whatever it is;
    the keys and values of its own positions, and of all of the shared pages, have to be finite (a NaN among them reaches any row of the
    sequence). 16-bit, dim a multiple of 8 up to 256."""
    if out is None and not _THROUGH_DISPATCHER:
        y = _front.paged_attention(q, k_pages, v_pages, page_table, lengths, starts, sm_scale, shared_pages)
        if y is not None:
            return y
    name = "paged_attention"
    if q.dtype not in (torch.float16, torch.bfloat16) or k_pages.dtype != q.dtype:
        raise TypeError("hexmi.paged_attention: queries and pages must both be float16 or both bfloat16")
    if q.dim() != 3 or k_pages.dim() != 4 or q.shape[2] != k_pages.shape[3] or q.shape[1] < 1 or q.shape[1] % max(k_pages.shape[1], 1) != 0:
        raise ValueError("hexmi.paged_attention: q is [tokens, heads, dim], the pages [pages, kv heads, page size, dim], and kv heads "
                         "divides heads")
    if q.shape[2] % 8 != 0 or q.shape[2] > 256:
        raise ValueError("hexmi.paged_attention: dim must be a multiple of 8 up to 256")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[2])
    if not 0 < sm_scale <= 2e38:
        raise ValueError("hexmi.paged_attention: sm_scale must be positive")
    if shared_pages is not None and (shared_pages.dtype != torch.int32 or shared_pages.dim() != 1 or shared_pages.shape[0] > page_table.shape[-1]):
        raise ValueError("hexmi.paged_attention: shared_pages must be an int32 tensor of one dimension, no longer than the table is wide")
    table, lens, begin = _paged_operands(name, q.shape[0], k_pages, v_pages, page_table, lengths, starts)
    dev = k_pages.device
    _one_device(name, dev, q, shared_pages, out)
    qd = _rows_of_heads(q, dev)
    if qd.data_ptr() % 16 or any(s % 8 for s in _strides(qd)[:2]):
        qd = qd.clone(memory_format=torch.contiguous_format)
    sd = _stage(shared_pages, dev)
    od = _out_like(out, q.shape, q.dtype, dev)
    read = [t for t in (qd, k_pages, v_pages, table, lens, begin, sd) if t is not None and t.numel()]
    if out is not None and od is out and od.numel() and (od.data_ptr() % 16 or _overlaps(od, *read)):
        od = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if q.shape[0]:
        args = (qd, k_pages, v_pages, table, lens, begin, float(sm_scale), sd, od)
        _run(name, _paged_attention_impl, args, *args)
    return _finish(od, out)


# Above this much multiply-add work the one-launch kernel (32 rows per workgroup, so few workgroups on small
# problems, and scalar guarded copies) loses to add -> tiled GEMM -> softmax: measured 5.9 us against 6.2 us at
# 32x32x32, 29 us against 10 us at 512x512x64. Below it the two saved launches and round trips win.
_FUSED_MAX_MACS = 1 << 20


def add_matmul_softmax(x, y, z, out=None, fused=None):
    """softmax((x + y) @ z, dim=-1): the graph of test/python/torch-mlir/test_add_matmul_softmax.py:19-29, which the
    reference compiles into one fused kernel. One launch (`hexmi_add_matmul_softmax`) when the result has at most
    1024 columns and the product is small; otherwise the three kernels run back to back on one stream.
    fused=True / False forces one or the other."""
    if x.shape != y.shape or x.dim() != 2 or z.dim() != 2 or x.shape[1] != z.shape[0]:
        raise ValueError("hexmi.add_matmul_softmax: x, y [M,K] and z [K,N] required")
    if not (x.dtype == y.dtype == z.dtype) or x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("hexmi.add_matmul_softmax: x, y, z must share one of float16, bfloat16, float32")
    dev = _device() if x.device.type != "cuda" else x.device
    M, K = x.shape
    N = z.shape[1]
    fits = 0 < N <= _lib.lib().hexmi_add_matmul_softmax_max_n()
    if fused is None:
        fused = fits and M * N * K <= _FUSED_MAX_MACS
    if fused:
        if not fits:
            raise ValueError("hexmi.add_matmul_softmax: the one-launch kernel takes at most 1024 columns")
        od = _out_like(out, (M, N), x.dtype, dev)
        _add_matmul_softmax_impl(_stage(x, dev), _stage(y, dev), _stage(z, dev), od)
        return _finish(od, out)
    total = binary("add", _stage(x, dev), _stage(y, dev))
    product = matmul(total, _stage(z, dev))
    return softmax(product, out=out)
