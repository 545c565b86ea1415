"""A cache in pages for requests that fork, over device buffers: the pages' changes of hands, their compaction, the
landing of new tokens in 8 bits with a scale per page and head, attention over them (include/sslm_hip.h has the
arithmetic, the layouts and the refusals).

As in batch_ops, buffers are device addresses, each method binds them once and returns a Call, and calling that with a
stream (None: the default stream) enqueues the operator on the buffers' present contents."""
from __future__ import annotations

import ctypes

from .batch_ops import BatchOps, Call
from .sslm import SslmLib

_I32, _I64, _U32, _P, _SZ = ctypes.c_int32, ctypes.c_int64, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_size_t

_POOL = [("pool", _P), ("page_bytes", _I64)]
_LAYER = _POOL + [("k_offset", _I64), ("v_offset", _I64), ("exp_offset", _I64), ("tables", _P), ("row_tokens", _P), ("row_start", _P)]


class CacheUpdateArgs(ctypes.Structure):
    """sslm_hip_cache_update_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("pages", _I32), ("page_tokens", _I32), ("table_ld", _I32),
                ("reserved", _I32)] + _POOL + [("tables", _P), ("lengths", _P), ("source", _P), ("keep", _P), ("room", _P),
                ("held", _P), ("new_tables", _P), ("new_lengths", _P), ("result", _P)]


class CacheCompactArgs(ctypes.Structure):
    """sslm_hip_cache_compact_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("pages", _I32), ("page_tokens", _I32), ("table_ld", _I32),
                ("reserved", _I32)] + _POOL + [("tables", _P), ("lengths", _P), ("held", _P), ("new_tables", _P), ("map", _P),
                ("result", _P)]


class CacheStoreArgs(ctypes.Structure):
    """sslm_hip_cache_store_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("tokens", _I32), ("max_new", _I32), ("heads", _I32), ("kv_heads", _I32),
                ("head_dim", _I32), ("pages", _I32), ("page_tokens", _I32), ("table_ld", _I32), ("rope_dim", _I32),
                ("rope_halves", _I32)] + _LAYER + [("rope_rows", _I64), ("rope_cos", _P), ("rope_sin", _P), ("q", _P), ("k", _P),
                ("v", _P), ("q_ld", _I64), ("k_ld", _I64), ("v_ld", _I64), ("k_scale", _P), ("v_scale", _P), ("r_t_k", _P),
                ("e_t_k", _P), ("r_t_v", _P), ("e_t_v", _P), ("q_out", _P), ("clamped", _P), ("status", _P)]


class CacheAttentionArgs(ctypes.Structure):
    """sslm_hip_cache_attention_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("tokens", _I32), ("max_new", _I32), ("heads", _I32), ("kv_heads", _I32),
                ("head_dim", _I32), ("pages", _I32), ("page_tokens", _I32), ("table_ld", _I32), ("reserved", _I32),
                ("max_width", _I64)] + _LAYER + [("q", _P), ("q_scale", _P), ("khead_m", _P), ("khead_e", _P), ("ln2_q", _I64),
                ("b_q", _I64), ("ca_q", _I64), ("ctx_fold", _P), ("site_m", _I64), ("site_e", _I64), ("codes", _P),
                ("scales", _P), ("status", _P)]


class StoreCall(Call):
    """sslm_hip_cache_store needs no workspace."""

    def __call__(self, stream: int | None = None, raw: bool = False):
        st = self._fn(self._ref, stream)
        if raw:
            return st
        if st:
            self._lib.check(self._name, st)


class CacheOps:
    def __init__(self, lib: SslmLib):
        self.lib = lib
        L = lib.lib
        for name, struct in (("update", CacheUpdateArgs), ("compact", CacheCompactArgs), ("attention", CacheAttentionArgs)):
            f = getattr(L, f"sslm_hip_cache_{name}")
            f.restype, f.argtypes = ctypes.c_int, [ctypes.POINTER(struct), _P, _SZ, _P]
            getattr(L, f"sslm_hip_cache_{name}_workspace").restype = _SZ
        L.sslm_hip_cache_store.restype, L.sslm_hip_cache_store.argtypes = ctypes.c_int, [ctypes.POINTER(CacheStoreArgs), _P]
        L.sslm_hip_cache_update_workspace.argtypes = L.sslm_hip_cache_compact_workspace.argtypes = [_I32] * 3
        L.sslm_hip_cache_attention_workspace.argtypes = [_I32] * 7 + [_I64]

    def update_workspace(self, rows, pages, table_ld) -> int:
        return self.lib.lib.sslm_hip_cache_update_workspace(rows, pages, table_ld)

    def update(self, *, workspace, workspace_bytes, **fields) -> Call:
        """sslm_hip_cache_update; the other keywords are CacheUpdateArgs' fields."""
        return Call(self.lib, "sslm_hip_cache_update", BatchOps._fill(CacheUpdateArgs(), fields), workspace, workspace_bytes)

    def compact_workspace(self, rows, pages, table_ld) -> int:
        return self.lib.lib.sslm_hip_cache_compact_workspace(rows, pages, table_ld)

    def compact(self, *, workspace, workspace_bytes, **fields) -> Call:
        """sslm_hip_cache_compact; the other keywords are CacheCompactArgs' fields."""
        return Call(self.lib, "sslm_hip_cache_compact", BatchOps._fill(CacheCompactArgs(), fields), workspace, workspace_bytes)

    def store(self, *, heads, kv_heads, head_dim, q_ld=None, k_ld=None, v_ld=None, **fields) -> StoreCall:
        """sslm_hip_cache_store; the other keywords are CacheStoreArgs' fields, the strides default to whole rows."""
        args = BatchOps._fill(CacheStoreArgs(), dict(
            fields, heads=heads, kv_heads=kv_heads, head_dim=head_dim, q_ld=heads * head_dim if q_ld is None else q_ld,
            k_ld=kv_heads * head_dim if k_ld is None else k_ld, v_ld=kv_heads * head_dim if v_ld is None else v_ld))
        return StoreCall(self.lib, "sslm_hip_cache_store", args, None, 0)

    def attention_workspace(self, rows, tokens, max_new, heads, kv_heads, head_dim, page_tokens, max_width) -> int:
        return self.lib.lib.sslm_hip_cache_attention_workspace(rows, tokens, max_new, heads, kv_heads, head_dim, page_tokens,
                                                               max_width)

    def attention(self, *, workspace, workspace_bytes, site, **fields) -> Call:
        """sslm_hip_cache_attention; `site` = (m, e), the other keywords are CacheAttentionArgs' fields."""
        args = BatchOps._fill(CacheAttentionArgs(), dict(fields, site_m=site[0], site_e=site[1]))
        return Call(self.lib, "sslm_hip_cache_attention", args, workspace, workspace_bytes)
