"""Typed entry points on device tensors (torch is only the allocator here).

Each function passes raw device pointers and the current CUDA stream to the
C ABI; the arithmetic is libnelisp_cuda's.  Tensors must be contiguous CUDA
tensors of the stated dtype.
"""
from __future__ import annotations

import ctypes

from . import _lib as L


_ready = False


def _lib():
    """The library, with its context on the current torch device."""
    global _ready
    lib = L.load()
    if not _ready:
        import torch
        L.check(lib.nl_init(torch.cuda.current_device()))
        _ready = True
    return lib


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream(stream=None):
    """The cudaStream_t of STREAM, or of torch's current stream on the
    library's device (read raw: building a Stream object for it costs more
    than the rest of a call)."""
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


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

_ROWS = {"torch.float32": 0, "torch.bfloat16": 1}     # NL_F32, NL_BF16
_PAIRS = {"half": 0, "adjacent": 1}


def _rows(t, name, dtype=None):
    """The row stride of a 2-D CUDA tensor of rows (f32 or bf16)."""
    stride = t.stride()
    if not t.is_cuda or len(stride) != 2 or (stride[1] != 1 and t.shape[1] > 1) or \
            (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name}: expected CUDA rows (2-D, unit inner stride"
                         + (f", {dtype})" if dtype is not None else ")"))
    return stride[0]


def _row_type(t):
    code = _ROWS.get(str(t.dtype))
    if code is None:
        raise ValueError(f"expected f32 or bf16 rows, not {t.dtype}")
    return code


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _workspace(nbytes, workspace, device, stream):
    """WORKSPACE as given, or one of the caching allocator that belongs to the
    call's stream, so that calls on different streams never share one."""
    import torch
    if workspace is not None:
        return workspace, workspace.numel() * workspace.element_size()
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _qk_shapes(QKV, GQ, GK, CO, SI, POS, Q, K, pairs):
    for t in (GQ, GK, CO, SI):
        _check_tensor(t, "torch.float32")
    _check_tensor(POS, "torch.int32")
    hd, n = GQ.numel(), QKV.shape[0]
    _need(hd > 0 and GK.numel() == hd, f"gains of {hd} and {GK.numel()} values")
    _need(CO.dim() == 2 and CO.shape == SI.shape, "CO and SI: two tables of one 2-D shape")
    _need(POS.numel() == n and Q.shape[0] == n and K.shape[0] == n,
          f"{n} rows of QKV, {POS.numel()} positions, {Q.shape[0]} and {K.shape[0]} rows")
    _need(Q.shape[1] % hd == 0 and K.shape[1] % hd == 0 and
          Q.shape[1] + K.shape[1] <= QKV.shape[1],
          f"rows of {QKV.shape[1]} values do not hold heads of {hd}: {Q.shape[1]} + {K.shape[1]}")
    _need(pairs in _PAIRS, f"pairs {pairs!r}: 'half' or 'adjacent'")
    return (n, Q.shape[1] // hd, K.shape[1] // hd, hd, 2 * CO.shape[1], CO.shape[0],
            _PAIRS[pairs])


def qk_norm_rope(QKV, GQ, GK, CO, SI, POS, Q, K, eps=1e-5, pairs="half", stream=None):
    """Q and K [n, heads * hd] and [n, kv_heads * hd] from the rows of QKV
    ([n, >= q | k]): each head's RMS norm with its gain (GQ, GK f32 [hd]) and
    the rotation of its first 2 * CO.shape[1] values at row POS[i] (int32) of
    the tables CO, SI.  Rows whose position is outside the tables are zeros.
    f32 or bf16; rows may be strided, and Q and K views of QKV itself."""
    dims = _qk_shapes(QKV, GQ, GK, CO, SI, POS, Q, K, pairs)
    xs = _rows(QKV, "QKV")
    qs, ks = _rows(Q, "Q", QKV.dtype), _rows(K, "K", QKV.dtype)
    L.check(_lib().nl_qk_norm_rope_dev(
        _row_type(QKV), QKV.data_ptr(), xs, GQ.data_ptr(), GK.data_ptr(), CO.data_ptr(),
        SI.data_ptr(), POS.data_ptr(), Q.data_ptr(), qs, K.data_ptr(), ks, *dims, eps,
        _stream(stream)))


def qk_norm_rope_bwd(QKV, GQ, GK, CO, SI, POS, DQ, DK, DQKV, DGQ, DGK, eps=1e-5, pairs="half",
                     workspace=None, stream=None):
    """The backward pass of qk_norm_rope: the q and k part of DQKV and the
    gains' gradients DGQ, DGK (f32 [hd]) from the gradients DQ, DK."""
    dims = _qk_shapes(QKV, GQ, GK, CO, SI, POS, DQ, DK, pairs)
    _check_tensor(DGQ, "torch.float32"); _check_tensor(DGK, "torch.float32")
    _need(DGQ.numel() == dims[3] and DGK.numel() == dims[3], "DGQ and DGK: one value per gain")
    _need(DQKV.shape[0] == dims[0] and DQKV.shape[1] >= DQ.shape[1] + DK.shape[1],
          f"DQKV of {tuple(DQKV.shape)} for {dims[0]} rows")
    xs, dxs = _rows(QKV, "QKV"), _rows(DQKV, "DQKV", QKV.dtype)
    qs, ks = _rows(DQ, "DQ", QKV.dtype), _rows(DK, "DK", QKV.dtype)
    lib = _lib()
    ws, nbytes = _workspace(lib.nl_qk_norm_rope_bwd_workspace_bytes(dims[3]), workspace,
                            QKV.device, stream)
    L.check(lib.nl_qk_norm_rope_bwd_dev(
        _row_type(QKV), QKV.data_ptr(), xs, GQ.data_ptr(), GK.data_ptr(), CO.data_ptr(),
        SI.data_ptr(), POS.data_ptr(), DQ.data_ptr(), qs, DK.data_ptr(), ks, DQKV.data_ptr(), dxs,
        DGQ.data_ptr(), DGK.data_ptr(), *dims, eps, ws.data_ptr(), nbytes, _stream(stream)))


def kv_cache(num_blocks, block_size, kv_heads, head_dim, bits, device="cuda"):
    """The four arrays of a quantised paged cache (8 or 4 bits a value), zeroed:
    KC, KP, VC, VP, the codes uint8 and the parameter words int32."""
    import torch
    _need(bits in (4, 8), f"bits {bits}: 8 or 4")
    shape = (num_blocks, kv_heads, block_size)
    KC, VC = (torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device)
              for _ in range(2))
    KP, VP = (torch.zeros(*shape, dtype=torch.int32, device=device) for _ in range(2))
    return KC, KP, VC, VP


def _pool(KC, KP, VC, VP, head_dim=None):
    """(bits, kv_heads, head_dim, block_size, num_blocks) of a cache."""
    shape = KC.shape
    for c, w in ((KC, KP), (VC, VP)):
        _check_tensor(c, "torch.uint8"); _check_tensor(w, "torch.int32")
        _need(len(shape) == 4 and c.shape == shape and w.shape == shape[:3],
              f"cache codes of {tuple(c.shape)} and words of {tuple(w.shape)}")
    bits = 8 * shape[3] // head_dim if head_dim else 0
    _need(bits in (4, 8) and bits * head_dim == 8 * shape[3],
          f"rows of {shape[3]} bytes for heads of {head_dim}")
    return bits, shape[1], head_dim, shape[2], shape[0]


def _kv_call(name, SLOT, KC, KP, VC, VP, K, V):
    _need(KC.dim() == 4, f"{name}: cache codes have 4 dimensions")
    width, kvh = K.shape[1], KC.shape[1]
    _need(kvh > 0 and width % kvh == 0 and V.shape == K.shape,
          f"{name}: rows of {width} values and {tuple(V.shape)} for {kvh} key heads")
    _check_tensor(SLOT, "torch.int32")
    _need(SLOT.numel() == K.shape[0], f"{name}: {SLOT.numel()} slots for {K.shape[0]} rows")
    return _pool(KC, KP, VC, VP, width // kvh)


def kv_append(K, V, SLOT, KC, KP, VC, VP, stream=None):
    """Quantise the rows K and V ([n, kv_heads * hd], f32 or bf16, may be
    strided) into the cache's token slots SLOT (int32 [n]; outside: skipped)."""
    bits, *dims = _kv_call("kv_append", SLOT, KC, KP, VC, VP, K, V)
    ks, vs = _rows(K, "K"), _rows(V, "V", K.dtype)
    L.check(_lib().nl_kv_append_dev(
        bits, _row_type(K), K.data_ptr(), ks, V.data_ptr(), vs, SLOT.data_ptr(), KC.data_ptr(),
        KP.data_ptr(), VC.data_ptr(), VP.data_ptr(), K.shape[0], *dims, _stream(stream)))


def kv_read(SLOT, KC, KP, VC, VP, K, V, stream=None):
    """The values of the slots SLOT into the rows K and V (outside: zeros)."""
    bits, *dims = _kv_call("kv_read", SLOT, KC, KP, VC, VP, K, V)
    ks, vs = _rows(K, "K"), _rows(V, "V", K.dtype)
    L.check(_lib().nl_kv_read_dev(
        bits, _row_type(K), SLOT.data_ptr(), KC.data_ptr(), KP.data_ptr(), VC.data_ptr(),
        VP.data_ptr(), K.data_ptr(), ks, V.data_ptr(), vs, K.shape[0], *dims, _stream(stream)))


def kv_move(SRC, DST, KC, KP, VC, VP, head_dim, stream=None):
    """Move tokens between slots without requantising them: SRC, DST int32
    [batch, count]; per sequence every source is read before any write."""
    _check_tensor(SRC, "torch.int32"); _check_tensor(DST, "torch.int32")
    _need(SRC.dim() == 2 and SRC.shape == DST.shape, "SRC and DST: [batch, count] each")
    bits, *dims = _pool(KC, KP, VC, VP, head_dim)
    L.check(_lib().nl_kv_move_dev(
        bits, SRC.data_ptr(), DST.data_ptr(), KC.data_ptr(), KP.data_ptr(), VC.data_ptr(),
        VP.data_ptr(), SRC.shape[0], SRC.shape[1], *dims, _stream(stream)))


def tree_attn(Q, KC, KP, VC, VP, TABLE, LEN, MASK, O, head_dim, scale=None, lse=None,
              workspace=None, stream=None):
    """Attention of MASK.shape[1] drafted tokens for each of MASK.shape[0]
    sequences over the quantised cache.  Q and O are rows (sequence, node) of
    heads * head_dim; TABLE int32 [batch, max_blocks]; LEN int32 [batch], the
    prefix tokens; MASK int64 [batch, nodes], bit j of node i set where i
    attends to node j (token LEN + j), 0 for an unused node.  SCALE is
    1/sqrt(head_dim) unless given; LSE (f32 [batch * nodes, heads]) receives
    the log of the softmax sums."""
    _check_tensor(TABLE, "torch.int32"); _check_tensor(LEN, "torch.int32")
    _check_tensor(MASK, "torch.int64"); _check_tensor(lse, "torch.float32")
    _need(MASK.dim() == 2 and TABLE.dim() == 2, "MASK and TABLE have 2 dimensions")
    batch, nodes = MASK.shape
    bits, kvh, hd, block_size, num_blocks = _pool(KC, KP, VC, VP, head_dim)
    qs, os_ = _rows(Q, "Q"), _rows(O, "O", Q.dtype)
    rows, width = Q.shape
    _need(LEN.numel() == batch and TABLE.shape[0] == batch and rows == batch * nodes and
          O.shape == Q.shape,
          f"tree_attn: {rows} rows, {batch} sequences of {nodes} nodes, {LEN.numel()} lengths, "
          f"a table of {tuple(TABLE.shape)}, outputs of {tuple(O.shape)}")
    heads = width // hd
    _need(width == heads * hd and (lse is None or lse.shape == (rows, heads)),
          f"tree_attn: rows of {width} values, heads of {hd}")
    lib = _lib()
    ws, nbytes = _workspace(lib.nl_tree_attn_workspace_bytes(nodes, heads, kvh, hd), workspace,
                            Q.device, stream)
    L.check(lib.nl_tree_attn_dev(
        bits, _row_type(Q), Q.data_ptr(), qs, KC.data_ptr(), KP.data_ptr(), VC.data_ptr(),
        VP.data_ptr(), TABLE.data_ptr(), LEN.data_ptr(), MASK.data_ptr(), O.data_ptr(), os_,
        lse.data_ptr() if lse is not None else None, batch, nodes, heads, kvh, hd, block_size,
        num_blocks, TABLE.shape[1], scale if scale is not None else hd ** -0.5, ws.data_ptr(),
        nbytes, _stream(stream)))


def launch_count() -> int:
    return int(L.load().nl_launch_count())
