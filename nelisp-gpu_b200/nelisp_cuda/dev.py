"""Typed entry points on device tensors (torch is only the allocator here).

Each function passes raw device pointers and the current CUDA stream to the
C ABI; the arithmetic is libnelisp_cuda's.  Tensors must be contiguous CUDA
tensors of the stated dtype.
"""
from __future__ import annotations

import ctypes

from . import _lib as L


_ready = None
_device = 0
_raw_stream = None


def _lib():
    """The library, with its context on the current torch device."""
    global _ready, _device, _raw_stream
    if _ready is None:
        import torch
        lib = L.load()
        L.check(lib.nl_init(torch.cuda.current_device()))
        _device = lib.nl_device()
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda device: torch.cuda.current_stream(device).cuda_stream)
        _ready = lib
    return _ready


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream(stream=None):
    """The cudaStream_t of STREAM, or of torch's current stream on the
    library's device (read raw: building a Stream object for it costs more
    than the rest of a call)."""
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        _lib()
    return _raw_stream(_device)


def _check_tensor(t, dtype_name):
    if t is None:
        return
    if not t.is_cuda or not t.is_contiguous() or str(t.dtype) != dtype_name:
        raise ValueError(f"expected a contiguous CUDA {dtype_name} tensor")


def dispatch(name, bufs, push, groups, stream=None):
    """Any registry kernel (a reference DSL name) on device tensors; the
    32-bit word count of each tensor is its bounds for the checks."""
    lib = _lib()
    n = len(bufs)
    ptrs = (ctypes.c_void_p * max(n, 1))(*[t.data_ptr() for t in bufs])
    words = (ctypes.c_uint32 * max(n, 1))(*[t.numel() * t.element_size() // 4 for t in bufs])
    L.check(lib.nl_dispatch_dev(name.encode(), n, ptrs, words, len(push), L.u32_array(push),
                                groups, _stream(stream)))


def ternary_workspace_bytes(seq: int, cols: int) -> int:
    return int(_lib().nl_ternary_workspace_bytes(seq, cols))


def ternary_rows(X, WP, BIAS, BETA, Y, seq, out, cols, nblk, wng, workspace=None, stream=None):
    _check_tensor(X, "torch.float32"); _check_tensor(Y, "torch.float32")
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    L.check(_lib().nl_ternary_rows_dev(_p(X), _p(WP), _p(BIAS), _p(BETA), _p(Y), seq, out,
                                         cols, nblk, wng, _p(workspace), ws_bytes,
                                         _stream(stream)))


def ternary_gemv(X, WP, S, Y, seq, out, cols, bias=None, workspace=None, stream=None):
    """Y = diag(S) (W X) (+ bias): per-row scales."""
    _check_tensor(X, "torch.float32"); _check_tensor(Y, "torch.float32")
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    L.check(_lib().nl_ternary_gemv_dev(_p(X), _p(WP), _p(S), _p(bias), _p(Y), seq, out, cols,
                                         _p(workspace), ws_bytes, _stream(stream)))


def ternary_gemv_batched(count, X, x_stride, WP, w_stride, S, s_stride, Y, y_stride, seq, out,
                         cols, workspace=None, stream=None):
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    L.check(_lib().nl_ternary_gemv_batched_dev(count, _p(X), x_stride, _p(WP), w_stride, _p(S),
                                                 s_stride, _p(Y), y_stride, seq, out, cols,
                                                 _p(workspace), ws_bytes, _stream(stream)))


def decode_attn_rope(QKV, CK, CV, POS, C, batch, heads, kv_heads, head_dim, max_seq,
                     rope_base=10000.0, stream=None):
    """One decode position: RoPE of q and the new key at POS[0] (int32 on the
    device), the cache append of key and value, attention over 0..POS[0]."""
    for t in (QKV, CK, CV, C):
        _check_tensor(t, "torch.float32")
    _check_tensor(POS, "torch.int32")
    L.check(_lib().nl_decode_attn_rope_dev(_p(QKV), _p(CK), _p(CV), _p(POS), _p(C), batch, heads,
                                             kv_heads, head_dim, max_seq, rope_base,
                                             _stream(stream)))


# ---- speculative serving: Q/K norm + RoPE, quantised KV cache, tree attention ----
# Called once a layer a token: the tensors are checked and the arguments filled
# in C++ (csrc/nl_torch.cpp); a refusal is a ValueError.

_ENTRIES = ("nl_qk_norm_rope_dev", "nl_qk_norm_rope_bwd_workspace_bytes",
            "nl_qk_norm_rope_bwd_dev", "nl_kv_append_dev", "nl_kv_read_dev", "nl_kv_move_dev",
            "nl_tree_attn_workspace_bytes", "nl_tree_attn_dev")
_module = None


def _bind():
    lib = _lib()
    _module.bind(_device, tuple(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                                for name in _ENTRIES))


def _load_serving():
    global _module
    import torch  # noqa: F401  (its libraries are what the module links to)
    try:
        from . import _serving
    except ImportError as e:
        raise RuntimeError(f"nelisp_cuda._serving is not built (make -C nelisp-gpu_b200): {e}")
    _serving.binder(_bind)
    _module = _serving
    return _serving


def _on(stream, function, *args):
    """FUNCTION with STREAM, one of the library's device, as the current one."""
    import torch
    _lib()
    if stream.device_index != _device:
        raise ValueError(f"a stream of cuda:{stream.device_index}: the library's device is "
                         f"cuda:{_device}")
    with torch.cuda.stream(stream):
        return function(*args)


def qk_norm_rope(QKV, GQ, GK, CO, SI, POS, Q, K, eps=1e-5, pairs="half", stream=None):
    """Q and K [n, heads * hd] and [n, kv_heads * hd] from the rows of QKV
    ([n, >= q | k]): each head's RMS norm with its gain (GQ, GK f32 [hd]) and
    the rotation of its first 2 * CO.shape[1] values at row POS[i] (int32) of
    the tables CO, SI.  Rows whose position is outside the tables are zeros.
    f32 or bf16; rows may be strided, and Q and K views of QKV itself."""
    if stream is not None:
        return _on(stream, qk_norm_rope, QKV, GQ, GK, CO, SI, POS, Q, K, eps, pairs)
    rc = (_module or _load_serving()).qk_norm_rope(QKV, GQ, GK, CO, SI, POS, Q, K, eps, pairs)
    if rc:
        L.check(rc)


def qk_norm_rope_bwd(QKV, GQ, GK, CO, SI, POS, DQ, DK, DQKV, DGQ, DGK, eps=1e-5, pairs="half",
                     workspace=None, stream=None):
    """The backward pass of qk_norm_rope: the q and k part of DQKV and the
    gains' gradients DGQ, DGK (f32 [hd]) from the gradients DQ, DK."""
    if stream is not None:
        return _on(stream, qk_norm_rope_bwd, QKV, GQ, GK, CO, SI, POS, DQ, DK, DQKV, DGQ, DGK, eps,
                   pairs, workspace)
    rc = (_module or _load_serving()).qk_norm_rope_bwd(QKV, GQ, GK, CO, SI, POS, DQ, DK, DQKV, DGQ,
                                                       DGK, eps, pairs, workspace)
    if rc:
        L.check(rc)


def kv_cache(num_blocks, block_size, kv_heads, head_dim, bits, device="cuda"):
    """The four arrays of a quantised paged cache (8 or 4 bits a value), zeroed:
    KC, KP, VC, VP, the codes uint8 and the parameter words int32."""
    import torch
    if bits not in (4, 8):
        raise ValueError("bits: 8 or 4")
    shape = (num_blocks, kv_heads, block_size)
    KC, VC = (torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device)
              for _ in range(2))
    KP, VP = (torch.zeros(*shape, dtype=torch.int32, device=device) for _ in range(2))
    return KC, KP, VC, VP


def kv_append(K, V, SLOT, KC, KP, VC, VP, stream=None):
    """Quantise the rows K and V ([n, kv_heads * hd], f32 or bf16, may be
    strided) into the cache's token slots SLOT (int32 [n]; outside: skipped; those
    inside must differ, or a slot given twice holds a mixture)."""
    if stream is not None:
        return _on(stream, kv_append, K, V, SLOT, KC, KP, VC, VP)
    rc = (_module or _load_serving()).kv_append(K, V, SLOT, KC, KP, VC, VP)
    if rc:
        L.check(rc)


def kv_read(SLOT, KC, KP, VC, VP, K, V, stream=None):
    """The values of the slots SLOT into the rows K and V (outside: zeros)."""
    if stream is not None:
        return _on(stream, kv_read, SLOT, KC, KP, VC, VP, K, V)
    rc = (_module or _load_serving()).kv_read(SLOT, KC, KP, VC, VP, K, V)
    if rc:
        L.check(rc)


def kv_move(SRC, DST, KC, KP, VC, VP, head_dim, stream=None):
    """Move tokens between slots without requantising them: SRC, DST int32
    [batch, count]; per sequence every source is read before any write, and of
    pairs with one destination the last is kept."""
    if stream is not None:
        return _on(stream, kv_move, SRC, DST, KC, KP, VC, VP, head_dim)
    rc = (_module or _load_serving()).kv_move(SRC, DST, KC, KP, VC, VP, head_dim)
    if rc:
        L.check(rc)


def tree_attn(Q, KC, KP, VC, VP, TABLE, LEN, MASK, O, head_dim, scale=None, lse=None,
              workspace=None, stream=None):
    """Attention of MASK.shape[1] drafted tokens for each of MASK.shape[0]
    sequences over the quantised cache.  Q and O are rows (sequence, node) of
    heads * head_dim; TABLE int32 [batch, max_blocks]; LEN int32 [batch], the
    prefix tokens; MASK int64 [batch, nodes], bit j of node i set where i
    attends to node j (token LEN + j), 0 for an unused node.  SCALE is
    1/sqrt(head_dim) unless given; LSE (f32 [batch * nodes, heads]) receives
    the log of the softmax sums.  The workspace, unless given, is the caching
    allocator's on the call's stream."""
    if stream is not None:
        return _on(stream, tree_attn, Q, KC, KP, VC, VP, TABLE, LEN, MASK, O, head_dim, scale, lse,
                   workspace)
    rc = (_module or _load_serving()).tree_attn(Q, KC, KP, VC, VP, TABLE, LEN, MASK, O, head_dim,
                                                scale, lse, workspace)
    if rc:
        L.check(rc)


def launch_count() -> int:
    return int(L.load().nl_launch_count())
