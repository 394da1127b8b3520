"""A base in 4 bits: codes with one fp16 scale (and, optionally, minimum) per group of elements of a row, scored exhaustively.

    packed = q4_pack(base_t, group=32)             # an eighth of the fp32 bytes, and the scales
    scores = q4_score(queries_t, packed)           # [nq, nb] fp32 inner products
    rows = q4_unpack(packed, ids)                  # fp32 values of some rows, for an exact re-score

Thin host layer over the C ABI (rg_q4_*, include/rg.h); everything is torch CUDA tensors, enqueued on the current stream.
"""
from collections import namedtuple

from ._lib import check, lib
from .softmax import _counts, _device, _dtype_code, _ptr, _rows, _stream, _stride

# codes uint8 [nb, >= ceil(dim / 8) * 4], scales fp16 [nb, ceil(dim / group)], mins alike or None (rg.h: "a base in 4 bits")
Q4Base = namedtuple("Q4Base", "codes scales mins dim group")


def _check_group(group):
    if group not in (32, 64, 128):
        raise ValueError("groups of 32, 64 or 128 elements")


def _check_form(p):
    import torch
    _check_group(p.group)
    groups = -(-p.dim // p.group)
    nb = p.codes.shape[0]
    if p.codes.dtype != torch.uint8 or p.codes.dim() != 2 or p.codes.stride(1) != 1 or not p.codes.is_cuda:
        raise ValueError("codes: rows of uint8 on a GPU are wanted")
    _counts(p.codes, "codes")
    if p.codes.shape[1] < -(-p.dim // 8) * 4:
        raise ValueError("codes: %d bytes a row, dim %d needs %d" % (p.codes.shape[1], p.dim, -(-p.dim // 8) * 4))
    if nb > 1 and p.codes.stride(0) < p.codes.shape[1]:
        raise ValueError("codes: rows that do not overlap are wanted, got strides %s" % (p.codes.stride(),))
    for t, name in ((p.scales, "scales"), (p.mins, "mins")):
        if t is None and name == "mins":
            continue
        if t.dtype != torch.float16 or t.shape != (nb, groups) or t.device != p.codes.device or (groups > 1 and t.stride(1) != 1):
            raise ValueError("%s: fp16 [%d, %d] on %s is wanted" % (name, nb, groups, p.codes.device))
        if nb > 1 and t.stride(0) < groups:
            raise ValueError("%s: rows that do not overlap are wanted, got strides %s" % (name, t.stride()))
    if p.mins is not None and nb > 1 and p.mins.stride(0) != p.scales.stride(0):
        raise ValueError("scales and mins have one row stride")


def q4_pack(base_t, group=32, mins=False):
    """rg_q4_pack_dev: rows (fp32 / fp16 / bf16) -> Q4Base."""
    import torch
    base_t = _rows(base_t, "base")
    code = _dtype_code(base_t)
    nb, dim = base_t.shape
    if not base_t.is_cuda:
        raise ValueError("base: a tensor on a GPU is wanted, got one on %s" % base_t.device)
    _check_group(group)
    groups = -(-dim // group)
    codes = torch.empty((nb, -(-dim // 8) * 4), dtype=torch.uint8, device=base_t.device)
    both = torch.empty((2 if mins else 1, nb, groups), dtype=torch.float16, device=base_t.device)
    low = both[1] if mins else None
    check(lib().rg_q4_pack_dev(_ptr(base_t), nb, _stride(base_t), dim, code, group, _ptr(codes),
                               codes.shape[1], _ptr(both[0]), _ptr(low), groups, _device(base_t), _stream(base_t)))
    return Q4Base(codes, both[0], low, dim, group)


def q4_unpack(packed, ids=None):
    """rg_q4_unpack_dev: fp32 values of all rows, or of the rows `ids` (int32 / int64 on the GPU; an id that is no row gives NaN)."""
    import torch
    _check_form(packed)
    nb = packed.codes.shape[0]
    if ids is not None:
        if ids.dim() != 1 or ids.device != packed.codes.device or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError("ids: a vector of int32 or int64 on %s is wanted" % packed.codes.device)
        _counts(ids, "ids")
        if ids.dtype == torch.int64:
            ids = ids.clamp(-1, 0xffffffff).to(torch.int32)      # (what 32 bits cannot say becomes an id that is no row)
        ids = ids.contiguous()
    n = nb if ids is None else ids.shape[0]
    out = torch.empty((n, packed.dim), dtype=torch.float32, device=packed.codes.device)
    check(lib().rg_q4_unpack_dev(_ptr(packed.codes), _stride(packed.codes), _ptr(packed.scales), _ptr(packed.mins), _stride(packed.scales), nb,
                                 packed.dim, packed.group, _ptr(ids), n, _ptr(out), packed.dim,
                                 _device(out), _stream(out)))
    return out


def q4_score(queries_t, packed, out=None):
    """rg_q4_score_dev: inner products [nq, nb], fp32, of the queries (fp32 / fp16 / bf16) with every row."""
    import torch
    _check_form(packed)
    queries_t = _rows(queries_t, "queries")
    code = _dtype_code(queries_t)
    nq, nb = queries_t.shape[0], packed.codes.shape[0]
    if queries_t.shape[1] != packed.dim or queries_t.device != packed.codes.device:
        raise ValueError("queries: %d columns on %s are wanted, got %d on %s" % (packed.dim, packed.codes.device, queries_t.shape[1], queries_t.device))
    if out is None:
        out = torch.empty((nq, nb), dtype=torch.float32, device=queries_t.device)
    elif out.shape != (nq, nb) or out.dtype != torch.float32 or out.device != queries_t.device or (nb > 1 and out.stride(1) != 1) or (nq > 1 and out.stride(0) < nb):
        raise ValueError("out: fp32 rows [%d, %d] on %s are wanted" % (nq, nb, queries_t.device))
    check(lib().rg_q4_score_dev(_ptr(packed.codes), _stride(packed.codes), _ptr(packed.scales), _ptr(packed.mins), _stride(packed.scales), nb,
                                packed.dim, packed.group, _ptr(queries_t), nq, _stride(queries_t), code,
                                _ptr(out), _stride(out), _device(out), _stream(out)))
    return out
