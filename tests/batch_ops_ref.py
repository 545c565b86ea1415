"""The batch operators (superslm_amd/batch_ops.py) row by row on the host, from the oracle's 64- and
128-bit primitives: what the GPU tests compare against, bit for bit."""
import ctypes

import numpy as np

from oracle_bind import LoraProj, Scale, _p, i8p, i32p, i64p

PINNED = [int(x * 2 ** 30) for x in (0.6931471805599453, 1.353, 0.344 / 0.3585)]
SITE = (1518500250, -45)
POSITION_OVER_CAP, ROW_WIDTH, REFUSED, SCALE_MANTISSA, SCALE_DERIVATION = 9, 7, 20, 4, 23


def bind(lib):
    lib.or_combine_scale.argtypes, lib.or_combine_scale.restype = [Scale, Scale], Scale
    i64 = ctypes.c_int64
    lib.or_iexp_scale_constants.argtypes = [i64, i64, i64, ctypes.c_int, i64, ctypes.c_int, i64, ctypes.c_int] + [i64p] * 3
    lib.or_check_softmax_width.argtypes = [i64, i64, ctypes.c_size_t]
    lib.or_softmax_row_q15.argtypes = [i64p, ctypes.c_size_t, i64, i64, i64, i64p]
    lib.or_apply_fold.argtypes, lib.or_apply_fold.restype = [i64] + [ctypes.c_int32] * 3, i64
    lib.or_requant_chain.argtypes = [i64p, ctypes.c_size_t, ctypes.POINTER(Scale), ctypes.c_size_t, Scale, i8p,
                                     ctypes.POINTER(Scale)]
    return lib


def _fits(m):
    return -(1 << 31) <= m < 1 << 31


def row_constants(lib, q_scale, khead, width):
    """(status, (q_ln2, q_b, q_c)) of a (row, KV head)."""
    if not _fits(q_scale[0]) or not _fits(khead[0]):
        return SCALE_MANTISSA, None
    s = lib.or_combine_scale(Scale(*q_scale), Scale(*khead))
    if not _fits(s.m):
        return SCALE_MANTISSA, None
    out = [ctypes.c_int64() for _ in range(3)]
    if lib.or_iexp_scale_constants(s.m, s.e, PINNED[0], 30, PINNED[1], 30, PINNED[2], 30, *[ctypes.byref(x) for x in out]):
        return SCALE_DERIVATION, None
    c = tuple(x.value for x in out)
    return lib.or_check_softmax_width(c[1], c[2], width), c


def attention_row(lib, q, q_scale, khead, k, v, ctx_fold, site=SITE):
    """One row: q [heads, D], k and v [kv_heads, width, D].  (status, codes, scale)."""
    nh, d = q.shape
    nkv, width = k.shape[:2]
    wide = np.zeros((nh, d), np.int64)
    for h in range(nh):
        j = h // (nh // nkv)
        st, c = row_constants(lib, q_scale, khead[j], width)
        if st:
            return st, None, None
        scores = np.ascontiguousarray(k[j].astype(np.int64) @ q[h].astype(np.int64))
        probs = np.zeros(width, np.int64)
        if not lib.or_softmax_row_q15(_p(scores, i64p), width, *c, _p(probs, i64p)):
            return REFUSED, None, None
        for i, x in enumerate(probs @ v[j].astype(np.int64)):
            wide[h, i] = lib.or_apply_fold(int(x), *[int(y) for y in ctx_fold[h]])
    codes, out = np.zeros(nh * d, np.int8), Scale()
    row = np.ascontiguousarray(wide.reshape(-1))
    st = lib.or_requant_chain(_p(row, i64p), row.size, None, 0, Scale(*site), _p(codes, i8p), ctypes.byref(out))
    return st, codes, (out.m, out.e)


def lora_row(lib, x, in_scale, w, fold, adapter, site=SITE):
    """One projected row: `adapter` is (a, ufold, b, dfold) or None.  (status, codes, scale)."""
    n, k = w.shape
    codes, out, lo, rank = np.zeros(n, np.int8), Scale(), None, 0
    if adapter is not None:
        a, uf, b, df = adapter
        rank, lo = a.shape[0], LoraProj(_p(a, i8p), _p(b, i8p), _p(uf, i32p), _p(df, i32p))
    st = lib.or_project_row(_p(x, i8p), Scale(*in_scale), k, n, _p(w, i8p), _p(fold, i32p), None,
                            ctypes.byref(lo) if lo is not None else None, rank, Scale(*site), _p(codes, i8p),
                            ctypes.byref(out))
    return st, codes, (out.m, out.e)


def pick_row(logits, history, bias, mask, repetition, presence, frequency):
    """One row's (token, adjusted logits): Python's integers for every changed token."""
    v = len(logits)
    x = logits.astype(object)
    for j, c in zip(*np.unique(history, return_counts=True)):
        if 0 <= j < v:
            y = int(x[j])
            y = (y << 16) // repetition if y > 0 else (y * repetition) >> 16
            x[j] = y - presence - frequency * int(c)
    for j, b in bias:
        if 0 <= j < v:
            x[j] = int(x[j]) + int(b)
    y = np.array([min(max(int(t), -(1 << 31)), (1 << 31) - 1) for t in x], dtype=np.int64)
    legal = np.ones(v, bool) if mask is None else np.unpackbits(mask, bitorder="little")[:v].astype(bool)
    y[~legal] = -(1 << 31)
    return (int(np.argmax(np.where(legal, y, -(1 << 40)))) if legal.any() else -1), y.astype(np.int32)
