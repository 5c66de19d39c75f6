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
# These are called once a layer a token: their checks are written for the time
# they take.

_PAIRS = {"half": 0, "adjacent": 1}      # NL_PAIRS_HALF, NL_PAIRS_ADJACENT
_PACK_QK = L.PACKED["nl_qk_norm_rope_dev"].pack
_PACK_QK_BWD = L.PACKED["nl_qk_norm_rope_bwd_dev"].pack
_PACK_ROWS = L.PACKED["nl_kv_rows"].pack
_PACK_MOVE = L.PACKED["nl_kv_move_dev"].pack
_PACK_TREE = L.PACKED["nl_tree_attn_dev"].pack
_types = None


def _torch_types():
    """(f32, bf16, int32, int64, uint8, {row type: NL_F32 / NL_BF16})."""
    global _types
    if _types is None:
        import torch
        _types = (torch.float32, torch.bfloat16, torch.int32, torch.int64, torch.uint8,
                  {torch.float32: 0, torch.bfloat16: 1})
    return _types


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _flat(dtype, *tensors):
    """Whether all are contiguous CUDA tensors of DTYPE."""
    for t in tensors:
        if t.dtype is not dtype or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"expected a contiguous CUDA {dtype} tensor, not {t.dtype} "
                             f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _rows(dtype, *tensors):
    """Whether all are 2-D CUDA rows of DTYPE with unit inner stride; the
    tensors' row strides."""
    strides = []
    for t in tensors:
        stride = t.stride()
        if t.dtype is not dtype or not t.is_cuda or len(stride) != 2 or \
                (stride[1] != 1 and t.shape[1] > 1):
            raise ValueError(f"expected CUDA rows of {dtype} (2-D, unit inner stride), not "
                             f"{t.dtype} {tuple(t.shape)} with strides {stride} on {t.device}")
        strides.append(stride[0])
    return strides


def _row_type(t):
    code = _torch_types()[5].get(t.dtype)
    if code is None:
        raise ValueError(f"expected f32 or bf16 rows, not {t.dtype}")
    return code


def _workspace(nbytes, workspace, device, stream):
    """WORKSPACE as given, or one of the caching allocator that belongs to the
    call's stream, so that calls on different streams never share one."""
    if workspace is not None:
        return workspace, workspace.numel() * workspace.element_size()
    import torch
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _qk_shapes(QKV, GQ, GK, CO, SI, POS, Q, K, pairs):
    types = _torch_types()
    _flat(types[0], GQ, GK, CO, SI)
    _flat(types[2], POS)
    (n, width), (nq, wq), (nk, wk) = QKV.shape, Q.shape, K.shape
    hd, table = GQ.numel(), CO.shape
    _need(hd > 0 and GK.numel() == hd, "gains of different or no length")
    _need(len(table) == 2 and table == SI.shape, "CO and SI: two tables of one 2-D shape")
    if POS.numel() != n or nq != n or nk != n:
        raise ValueError(f"{n} rows of QKV, {POS.numel()} positions, {nq} and {nk} rows")
    if wq % hd or wk % hd or wq + wk > width:
        raise ValueError(f"rows of {width} values do not hold heads of {hd}: {wq} + {wk}")
    _need(pairs in _PAIRS, "pairs: 'half' or 'adjacent'")
    return n, wq // hd, wk // hd, hd, 2 * table[1], table[0]


def qk_norm_rope(QKV, GQ, GK, CO, SI, POS, Q, K, eps=1e-5, pairs="half", stream=None):
    """Q and K [n, heads * hd] and [n, kv_heads * hd] from the rows of QKV
    ([n, >= q | k]): each head's RMS norm with its gain (GQ, GK f32 [hd]) and
    the rotation of its first 2 * CO.shape[1] values at row POS[i] (int32) of
    the tables CO, SI.  Rows whose position is outside the tables are zeros.
    f32 or bf16; rows may be strided, and Q and K views of QKV itself."""
    kind = _row_type(QKV)
    xs, qs, ks = _rows(QKV.dtype, QKV, Q, K)
    dims = _qk_shapes(QKV, GQ, GK, CO, SI, POS, Q, K, pairs)
    rc = _lib().nl_qk_norm_rope_dev(_PACK_QK(
        kind, _PAIRS[pairs], QKV.data_ptr(), xs, GQ.data_ptr(), GK.data_ptr(), CO.data_ptr(),
        SI.data_ptr(), POS.data_ptr(), Q.data_ptr(), qs, K.data_ptr(), ks, *dims, eps),
        _stream(stream))
    if rc:
        L.check(rc)


def qk_norm_rope_bwd(QKV, GQ, GK, CO, SI, POS, DQ, DK, DQKV, DGQ, DGK, eps=1e-5, pairs="half",
                     workspace=None, stream=None):
    """The backward pass of qk_norm_rope: the q and k part of DQKV and the
    gains' gradients DGQ, DGK (f32 [hd]) from the gradients DQ, DK."""
    kind = _row_type(QKV)
    xs, qs, ks, dxs = _rows(QKV.dtype, QKV, DQ, DK, DQKV)
    dims = _qk_shapes(QKV, GQ, GK, CO, SI, POS, DQ, DK, pairs)
    _flat(_torch_types()[0], DGQ, DGK)
    hd = dims[3]
    _need(DGQ.numel() == hd and DGK.numel() == hd, "DGQ and DGK: one value per gain")
    n, width = DQKV.shape
    if n != dims[0] or width < DQ.shape[1] + DK.shape[1]:
        raise ValueError(f"DQKV of {n} x {width} for {dims[0]} rows")
    lib = _lib()
    ws, nbytes = _workspace(lib.nl_qk_norm_rope_bwd_workspace_bytes(hd), workspace, QKV.device,
                            stream)
    rc = lib.nl_qk_norm_rope_bwd_dev(_PACK_QK_BWD(
        kind, _PAIRS[pairs], QKV.data_ptr(), xs, GQ.data_ptr(), GK.data_ptr(), CO.data_ptr(),
        SI.data_ptr(), POS.data_ptr(), DQ.data_ptr(), qs, DK.data_ptr(), ks, DQKV.data_ptr(), dxs,
        DGQ.data_ptr(), DGK.data_ptr(), *dims, eps, ws.data_ptr(), nbytes), _stream(stream))
    if rc:
        L.check(rc)


def kv_cache(num_blocks, block_size, kv_heads, head_dim, bits, device="cuda"):
    """The four arrays of a quantised paged cache (8 or 4 bits a value), zeroed:
    KC, KP, VC, VP, the codes uint8 and the parameter words int32."""
    import torch
    _need(bits in (4, 8), "bits: 8 or 4")
    shape = (num_blocks, kv_heads, block_size)
    KC, VC = (torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device)
              for _ in range(2))
    KP, VP = (torch.zeros(*shape, dtype=torch.int32, device=device) for _ in range(2))
    return KC, KP, VC, VP


def _pool(KC, KP, VC, VP, head_dim):
    """A cache as the fields of nl_kv_cache."""
    types = _torch_types()
    _flat(types[4], KC, VC)
    _flat(types[2], KP, VP)
    shape = KC.shape
    if len(shape) != 4 or VC.shape != shape or KP.shape != shape[:3] or VP.shape != shape[:3]:
        raise ValueError(f"cache codes of {tuple(shape)} and {tuple(VC.shape)}, words of "
                         f"{tuple(KP.shape)} and {tuple(VP.shape)}")
    blocks, kvh, size, row = shape
    if row == head_dim:
        bits = 8
    elif 2 * row == head_dim:
        bits = 4
    else:
        raise ValueError(f"rows of {row} bytes for heads of {head_dim}")
    return (bits, kvh, head_dim, size, blocks, KC.data_ptr(), KP.data_ptr(), VC.data_ptr(),
            VP.data_ptr())


def _kv_shapes(SLOT, KC, KP, VC, VP, K, V):
    _flat(_torch_types()[2], SLOT)
    _need(KC.dim() == 4, "cache codes have 4 dimensions")
    (n, width), kvh = K.shape, KC.shape[1]
    if V.shape != K.shape or SLOT.numel() != n or kvh == 0 or width % kvh:
        raise ValueError(f"rows of {n} x {width} and {tuple(V.shape)}, {SLOT.numel()} slots, "
                         f"{kvh} key heads")
    return n, _pool(KC, KP, VC, VP, width // kvh)


def kv_append(K, V, SLOT, KC, KP, VC, VP, stream=None):
    """Quantise the rows K and V ([n, kv_heads * hd], f32 or bf16, may be
    strided) into the cache's token slots SLOT (int32 [n]; outside: skipped)."""
    kind = _row_type(K)
    ks, vs = _rows(K.dtype, K, V)
    n, pool = _kv_shapes(SLOT, KC, KP, VC, VP, K, V)
    rc = _lib().nl_kv_append_dev(_PACK_ROWS(
        *pool, kind, n, SLOT.data_ptr(), K.data_ptr(), ks, V.data_ptr(), vs), _stream(stream))
    if rc:
        L.check(rc)


def kv_read(SLOT, KC, KP, VC, VP, K, V, stream=None):
    """The values of the slots SLOT into the rows K and V (outside: zeros)."""
    kind = _row_type(K)
    ks, vs = _rows(K.dtype, K, V)
    n, pool = _kv_shapes(SLOT, KC, KP, VC, VP, K, V)
    rc = _lib().nl_kv_read_dev(_PACK_ROWS(
        *pool, kind, n, SLOT.data_ptr(), K.data_ptr(), ks, V.data_ptr(), vs), _stream(stream))
    if rc:
        L.check(rc)


def kv_move(SRC, DST, KC, KP, VC, VP, head_dim, stream=None):
    """Move tokens between slots without requantising them: SRC, DST int32
    [batch, count]; per sequence every source is read before any write."""
    _flat(_torch_types()[2], SRC, DST)
    _need(SRC.dim() == 2 and SRC.shape == DST.shape, "SRC and DST: [batch, count] each")
    L.check(_lib().nl_kv_move_dev(_PACK_MOVE(
        *_pool(KC, KP, VC, VP, head_dim), SRC.data_ptr(), DST.data_ptr(), *SRC.shape),
        _stream(stream)))


def tree_attn(Q, KC, KP, VC, VP, TABLE, LEN, MASK, O, head_dim, scale=None, lse=None,
              workspace=None, stream=None):
    """Attention of MASK.shape[1] drafted tokens for each of MASK.shape[0]
    sequences over the quantised cache.  Q and O are rows (sequence, node) of
    heads * head_dim; TABLE int32 [batch, max_blocks]; LEN int32 [batch], the
    prefix tokens; MASK int64 [batch, nodes], bit j of node i set where i
    attends to node j (token LEN + j), 0 for an unused node.  SCALE is
    1/sqrt(head_dim) unless given; LSE (f32 [batch * nodes, heads]) receives
    the log of the softmax sums."""
    types = _torch_types()
    kind = _row_type(Q)
    qs, os_ = _rows(Q.dtype, Q, O)
    _flat(types[2], TABLE, LEN)
    _flat(types[3], MASK)
    pool = _pool(KC, KP, VC, VP, head_dim)
    table, mask, shape = TABLE.shape, MASK.shape, Q.shape
    _need(len(mask) == 2 and len(table) == 2, "MASK and TABLE have 2 dimensions")
    batch, nodes = mask
    rows, width = shape
    heads = width // head_dim
    if LEN.numel() != batch or table[0] != batch or rows != batch * nodes or O.shape != shape or \
            width != heads * head_dim:
        raise ValueError(f"tree_attn: {rows} rows of {width}, heads of {head_dim}, {batch} "
                         f"sequences of {nodes} nodes, {LEN.numel()} lengths, a table of "
                         f"{tuple(table)}, outputs of {tuple(O.shape)}")
    out_lse = 0
    if lse is not None:
        _flat(types[0], lse)
        _need(lse.shape == (rows, heads), "lse: a value per row and head")
        out_lse = lse.data_ptr()
    lib = _lib()
    ws, nbytes = _workspace(lib.nl_tree_attn_workspace_bytes(nodes, heads, pool[1], head_dim),
                            workspace, Q.device, stream)
    rc = lib.nl_tree_attn_dev(_PACK_TREE(
        *pool, kind, batch, nodes, heads, table[1],
        scale if scale is not None else head_dim ** -0.5, Q.data_ptr(), qs, TABLE.data_ptr(),
        LEN.data_ptr(), MASK.data_ptr(), O.data_ptr(), os_, out_lse, ws.data_ptr(), nbytes),
        _stream(stream))
    if rc:
        L.check(rc)


def launch_count() -> int:
    return int(L.load().nl_launch_count())
