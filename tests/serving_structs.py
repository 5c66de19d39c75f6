"""The argument structures of the serving entry points, for calling the C ABI
through ctypes: in the header's field order and the C compiler's layout."""
import struct

_CACHE = "iIIIIPPPP"           # nl_kv_cache
PACKED = {
    "nl_qk_norm_rope_dev": struct.Struct("@iiPQPPPPPPQPQIIIIIIf"),
    "nl_qk_norm_rope_bwd_dev": struct.Struct("@iiPQPPPPPPQPQPQPPIIIIIIfPN"),
    "nl_kv_rows": struct.Struct("@" + _CACHE + "iIPPQPQ"),
    "nl_kv_move_dev": struct.Struct("@" + _CACHE + "PPII"),
    "nl_tree_attn_dev": struct.Struct("@" + _CACHE + "iIIIIfPQPPPPQPPN"),
}
