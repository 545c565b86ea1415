"""The operators of a decode step whose rows are different requests, over device buffers: attention
of rows that share prompts, a projection with an adapter of its own per row, the next token under
each row's own rules (include/sslm_hip.h has the arithmetic, the layouts and the refusals).

Buffers are device addresses (a DeviceArray's `ptr`, another allocator's pointer in a process with one
HIP runtime).  Each method binds its buffers once and returns a Call; calling it with a stream (None:
the default stream) enqueues the operator on the buffers' present contents."""
from __future__ import annotations

import ctypes
from numbers import Integral

from .sslm import SslmLib

_I32, _I64, _U32, _P, _SZ = ctypes.c_int32, ctypes.c_int64, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_size_t


class SharedAttentionArgs(ctypes.Structure):
    """sslm_hip_shared_attention_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32),
                ("prefixes", _I32), ("blocks", _I32), ("reserved", _I32), ("max_prefix", _I64), ("max_own", _I64),
                ("kv_pool", _P), ("block_bytes", _I64), ("k_offset", _I64), ("v_offset", _I64), ("cap", _I64),
                ("q", _P), ("q_scale", _P), ("khead_m", _P), ("khead_e", _P), ("ln2_q", _I64), ("b_q", _I64),
                ("ca_q", _I64), ("ctx_fold", _P), ("site_m", _I64), ("site_e", _I64), ("row_block", _P),
                ("row_width", _P), ("prefix_rows", _P), ("prefix_block", _P), ("prefix_len", _P), ("codes", _P),
                ("scales", _P), ("status", _P)]


class Lora(ctypes.Structure):
    """sslm_hip_lora: one adapter of a batch."""
    _fields_ = [("a", _P), ("ufold", _P), ("b", _P), ("dfold", _P), ("rank", _I32), ("reserved", _I32)]


class GemmLoraArgs(ctypes.Structure):
    """sslm_hip_gemm_lora_args."""
    _fields_ = [("struct_size", _U32), ("m", _I32), ("n", _I32), ("k", _I32), ("adapter_count", _I32),
                ("reserved", _I32), ("a", _P), ("w", _P), ("fold", _P), ("in_scale", _P), ("site_m", _I64),
                ("site_e", _I64), ("adapters", _P), ("row_adapter", _P), ("codes", _P), ("scales", _P), ("status", _P)]


class LogitRule(ctypes.Structure):
    """sslm_hip_logit_rule: the rules of one row of logits."""
    _fields_ = [("history", _P), ("bias_ids", _P), ("bias_values", _P), ("mask", _P), ("history_len", _I32),
                ("bias_count", _I32), ("repetition_q16", _I32), ("presence", _I32), ("frequency", _I32),
                ("reserved", _I32)]


class PickArgs(ctypes.Structure):
    """sslm_hip_pick_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("vocab", _I32), ("reserved", _I32), ("logits", _P),
                ("logits_ld", _I64), ("adjusted_ld", _I64), ("rules", _P), ("adjusted", _P), ("tokens", _P)]


class Sampling(ctypes.Structure):
    """sslm_hip_sampling: how one row of logits is sampled."""
    _fields_ = [("mask", _P), ("q_ln2", _I64), ("q_b", _I64), ("q_c", _I64), ("top_k", _I32), ("top_p_q16", _I32),
                ("min_p_q16", _I32), ("random", _U32)]


class SampleArgs(ctypes.Structure):
    """sslm_hip_sample_args."""
    _fields_ = [("struct_size", _U32), ("rows", _I32), ("vocab", _I32), ("reserved", _I32), ("logits", _P),
                ("logits_ld", _I64), ("rules", _P), ("tokens", _P), ("mass", _P)]


def sampling_constants(unit: float) -> dict:
    """q_ln2, q_b and q_c for logits of which `unit` make one natural unit at the wanted temperature: the
    temperature over the real value of one integer step."""
    return {"q_ln2": int(0.6931471805599453 * unit), "q_b": int(1.353 * unit), "q_c": int(0.344 / 0.3585 * unit * unit)}


class Call:
    """One operator over bound buffers.  `args` is its struct, whose fields may be changed between calls."""

    def __init__(self, lib: SslmLib, name: str, args, workspace: int, workspace_bytes: int):
        self._lib, self._name, self.args = lib, name, args
        self._fn = getattr(lib.lib, name)
        self._ref, self._ws, self._bytes = ctypes.byref(args), workspace, workspace_bytes

    def __call__(self, stream: int | None = None, raw: bool = False):
        st = self._fn(self._ref, self._ws, self._bytes, stream)
        if raw:
            return st
        if st:
            self._lib.check(self._name, st)


class BatchOps:
    def __init__(self, lib: SslmLib):
        self.lib = lib
        L = lib.lib
        for name, struct in (("sslm_hip_shared_attention", SharedAttentionArgs),
                             ("sslm_hip_gemm_lora_requant", GemmLoraArgs), ("sslm_hip_pick_tokens", PickArgs),
                             ("sslm_hip_sample_tokens", SampleArgs)):
            f = getattr(L, name)
            f.restype, f.argtypes = ctypes.c_int, [ctypes.POINTER(struct), _P, _SZ, _P]
        L.sslm_hip_shared_attention_workspace.argtypes = [_I32] * 5 + [_I64] * 2
        L.sslm_hip_gemm_lora_workspace.argtypes = [_I32] * 3
        L.sslm_hip_pick_workspace.argtypes = L.sslm_hip_sample_workspace.argtypes = [_I32] * 2
        for name in ("shared_attention", "gemm_lora", "pick", "sample"):
            getattr(L, f"sslm_hip_{name}_workspace").restype = _SZ

    @staticmethod
    def _fill(args, fields):
        args.struct_size = ctypes.sizeof(args)
        for k, v in fields.items():
            if not hasattr(args, k):
                raise TypeError(f"{type(args).__name__} has no field {k}")
            setattr(args, k, v)
            if isinstance(v, Integral) and (getattr(args, k) or 0) != v:  # ctypes keeps the low bits alone
                raise OverflowError(f"{type(args).__name__}.{k} does not hold {v}")
        return args

    def shared_attention_workspace(self, rows, heads, kv_heads, head_dim, prefixes, max_prefix, max_own) -> int:
        return self.lib.lib.sslm_hip_shared_attention_workspace(rows, heads, kv_heads, head_dim, prefixes, max_prefix,
                                                                max_own)

    def shared_attention(self, *, workspace, workspace_bytes, site, **fields) -> Call:
        """sslm_hip_shared_attention; `site` = (m, e), the other keywords are SharedAttentionArgs' fields."""
        args = self._fill(SharedAttentionArgs(), dict(fields, site_m=site[0], site_e=site[1]))
        return Call(self.lib, "sslm_hip_shared_attention", args, workspace, workspace_bytes)

    def gemm_lora_workspace(self, m, n, k) -> int:
        return self.lib.lib.sslm_hip_gemm_lora_workspace(m, n, k)

    def gemm_lora_requant(self, *, workspace, workspace_bytes, site, **fields) -> Call:
        """sslm_hip_gemm_lora_requant; `site` = (m, e), the other keywords are GemmLoraArgs' fields."""
        args = self._fill(GemmLoraArgs(), dict(fields, site_m=site[0], site_e=site[1]))
        return Call(self.lib, "sslm_hip_gemm_lora_requant", args, workspace, workspace_bytes)

    def pick_workspace(self, rows, vocab) -> int:
        return self.lib.lib.sslm_hip_pick_workspace(rows, vocab)

    def pick_tokens(self, *, workspace, workspace_bytes, vocab, logits_ld=None, adjusted_ld=None, **fields) -> Call:
        """sslm_hip_pick_tokens; row strides default to the vocabulary."""
        args = self._fill(PickArgs(), dict(fields, vocab=vocab, logits_ld=vocab if logits_ld is None else logits_ld,
                                           adjusted_ld=vocab if adjusted_ld is None else adjusted_ld))
        return Call(self.lib, "sslm_hip_pick_tokens", args, workspace, workspace_bytes)

    def sample_workspace(self, rows, vocab) -> int:
        return self.lib.lib.sslm_hip_sample_workspace(rows, vocab)

    def sample_tokens(self, *, workspace, workspace_bytes, vocab, logits_ld=None, **fields) -> Call:
        """sslm_hip_sample_tokens; `rules` is a device array of Sampling, the row stride defaults to the vocabulary."""
        args = self._fill(SampleArgs(), dict(fields, vocab=vocab, logits_ld=vocab if logits_ld is None else logits_ld))
        return Call(self.lib, "sslm_hip_sample_tokens", args, workspace, workspace_bytes)
