"""A LoRA adapter artifact's tensors as arrays, for the oracle (OracleModel's `adapter`)."""
import struct

import numpy as np

from superslm_amd.sslm_artifact import HEADER_BYTES, SEC_DELTA_FOLD, SEC_PROVENANCE, SEC_U_FOLD, SEC_WEIGHTS, SECTION_DESC_BYTES


def _manifest(blob, base, dtype):
    count, names_len = struct.unpack_from("<II", blob, base + 8)
    names = base + 16 + 48 * count
    out = {}
    for i in range(count):
        off, length, nd, *rest = struct.unpack_from("<III4IQQI", blob, base + 16 + 48 * i)
        shape, at = rest[:nd], rest[4]
        n = int(np.prod(shape))
        out[blob[names + off:names + off + length].decode()] = np.frombuffer(blob, dtype, n, base + at).reshape(shape).copy()
    return out


class AdapterView:
    def __init__(self, blob):
        blob = bytes(blob)
        sections = {}
        for i in range(struct.unpack_from("<I", blob, 12)[0]):
            typ, _, off = struct.unpack_from("<IIQ", blob, HEADER_BYTES + i * SECTION_DESC_BYTES)
            sections[typ] = off
        self.rank = struct.unpack_from("<i", blob, sections[SEC_PROVENANCE] + 8)[0]
        w = _manifest(blob, sections[SEC_WEIGHTS], np.int8)
        self.a = {k[:-7]: v for k, v in w.items() if k.endswith(".lora_A")}
        self.b = {k[:-7]: v for k, v in w.items() if k.endswith(".lora_B")}
        self.d_fold = _manifest(blob, sections[SEC_DELTA_FOLD], np.int32)
        self.u_fold = _manifest(blob, sections[SEC_U_FOLD], np.int32)


def with_delta_exponent(blob, exponent):
    """The adapter with every delta fold row (identity 0, mult 2^30, `exponent`), its hash recomputed."""
    from superslm_amd.sslm_artifact import with_flags
    out = bytearray(blob)
    for i in range(struct.unpack_from("<I", out, 12)[0]):
        typ, _, off = struct.unpack_from("<IIQ", out, HEADER_BYTES + i * SECTION_DESC_BYTES)
        if typ != SEC_DELTA_FOLD:
            continue
        for k in range(struct.unpack_from("<I", out, off + 8)[0]):
            _, _, nd, *rest = struct.unpack_from("<III4IQQI", out, off + 16 + 48 * k)
            rows = np.frombuffer(out, np.int32, int(np.prod(rest[:nd])), off + rest[4]).reshape(-1, 3)
            rows[:] = (0, 1 << 30, exponent)
    return with_flags(bytes(out), struct.unpack_from("<I", out, 16)[0])
