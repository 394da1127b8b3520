"""Softmax cross entropy over ALL rows of a base: trains the tables and towers that the index serves.

    loss = softmax_loss(queries, base, targets, scale=1 / temperature)      # [nq] fp32, differentiable in queries and base
    loss.mean().backward()

queries [nq, dim] and base [nb, dim] are torch CUDA tensors of one dtype (fp32, fp16, bf16); targets [nq] holds the row of the base that
answers each query (e.g. column 0 of the ground truth; for cosine normalise the rows first), -1 where there is none (loss 0, no gradient).
The nq x nb logits are never stored.  Thin host layer over the C ABI (rg_softmax_*, include/rg.h); the multi-GPU form holds a row shard of
the base per rank, like the ground truth.
"""
import ctypes as C
import functools

from ._lib import check, lib

STATS, MEAN, GRAD = 0, 1, 2


_codes = {}


def _dtype_code(t):
    code = _codes.get(t.dtype)
    if code is None:
        import torch
        _codes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        code = _codes.get(t.dtype)
        if code is None:
            raise TypeError("rows are fp32, fp16 or bf16, got %s" % t.dtype)
    return code


def _counts(t, name):
    """sizes reach the C ABI in 32 bits, of which ctypes takes the lowest without a word"""
    if max(t.shape) > 0x7fffffff:
        raise ValueError("%s: at most 2^31 - 1 rows and columns, got shape %s" % (name, tuple(t.shape)))


def _id_base(n):
    if not 0 <= n <= 0xffffffff:
        raise ValueError("id_base: a row id of 32 bits is wanted, got %d" % n)
    return n


def _rows(t, name):
    """t itself where its rows can be read in place, else a contiguous copy (transposed or broadcast tensors)."""
    if t.dim() != 2:
        raise ValueError("%s: a matrix of rows is wanted, got shape %s" % (name, tuple(t.shape)))
    _counts(t, name)
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1] or t.is_contiguous():
        return t
    return t.contiguous()


def _stride(t):
    return max(t.stride(0), t.shape[1])     # (a single row's stride may be anything)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _stream(t):
    import torch
    return torch._C._cuda_getCurrentRawStream(t.device.index)     # (current_stream(...).cuda_stream without the objects: 2 us of a call)


def _device(t):
    return t.device.index or 0


def _check_pair(queries, base):
    if not queries.is_cuda or queries.device != base.device:
        raise ValueError("queries and base live on one GPU, got %s and %s" % (queries.device, base.device))
    if queries.dtype != base.dtype:
        raise TypeError("queries and base have one dtype, got %s and %s" % (queries.dtype, base.dtype))
    if queries.shape[1] != base.shape[1]:
        raise ValueError("queries have %d columns, the base has %d" % (queries.shape[1], base.shape[1]))


def _check_vector(t, n, dtype, like, name):
    if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype or t.device != like.device:
        raise ValueError("%s: %d values of %s on %s are wanted, got %s of %s on %s" % (name, n, dtype, like.device, tuple(t.shape), t.dtype, t.device))
    return t.contiguous()


def _targets(targets, n, like):
    """ids as 32 bits (of int64: -1 and ids up to 2^32 - 2 keep their meaning, what 32 bits cannot say becomes 2^32 - 2, which no base has)"""
    import torch
    if targets.dtype == torch.int64:
        targets = targets.clamp(-2, 0xfffffffe).to(torch.int32)
    return _check_vector(targets, n, torch.int32, like, "targets")


@functools.lru_cache(maxsize=1024)
def workspace(what, nb, nq, dim, dtype_code):
    """rg_softmax_workspace: bytes of scratch of one call"""
    if not 0 <= min(nb, nq, dim) <= max(nb, nq, dim) <= 0xffffffff:
        raise ValueError("sizes of 32 bits are wanted, got %d, %d, %d" % (nb, nq, dim))
    n = C.c_uint64()
    check(lib().rg_softmax_workspace(what, nb, nq, dim, dtype_code, C.byref(n)))
    return n.value


def _scratch(what, nb, nq, dim, like):
    import torch
    n = workspace(what, nb, nq, dim, _dtype_code(like))
    return like.new_empty(max(n, 256), dtype=torch.uint8), n


def softmax_shard_dev(base_t, queries_t, targets_t, scale, id_base=0, want_mean=False):
    """rg_softmax_shard_dev on the current stream: (rest, own, lse, loss, mean) of one row shard, fp32; lse and loss as if the shard were the
    whole base; mean is None unless asked for."""
    import torch
    queries_t, base_t, id_base = _rows(queries_t, "queries"), _rows(base_t, "base"), _id_base(id_base)
    _check_pair(queries_t, base_t)
    nq, nb, dim = queries_t.shape[0], base_t.shape[0], base_t.shape[1]
    targets_t = _targets(targets_t, nq, base_t)
    rest, own, lse, loss = torch.empty((4, nq), dtype=torch.float32, device=base_t.device).unbind(0)
    mean = torch.empty((nq, dim), dtype=torch.float32, device=base_t.device) if want_mean else None
    work, n = _scratch(MEAN if want_mean else STATS, nb, nq, dim, base_t)
    check(lib().rg_softmax_shard_dev(_ptr(base_t), nb, _stride(base_t), _ptr(queries_t), nq, _stride(queries_t),
                                     dim, _dtype_code(base_t), scale, _ptr(targets_t), id_base,
                                     _ptr(rest), _ptr(own), _ptr(lse), _ptr(loss), _ptr(mean), _ptr(work), n, _device(base_t),
                                     _stream(base_t)))
    return rest, own, lse, loss, mean


def softmax_merge_dev(rest_in, own_in, targets_t):
    """rg_softmax_merge_dev: statistics [nlists, nq] of the row shards -> (lse, loss) over the whole base."""
    import torch
    if rest_in.dim() != 2 or rest_in.shape != own_in.shape or rest_in.dtype != torch.float32 or own_in.dtype != torch.float32 or rest_in.device != own_in.device or not rest_in.is_cuda:
        raise ValueError("rest and own: two fp32 matrices [nlists, nq] on one GPU are wanted")
    _counts(rest_in, "rest and own")
    rest_in, own_in = rest_in.contiguous(), own_in.contiguous()
    targets_t = _targets(targets_t, rest_in.shape[1], rest_in)
    lse, loss = torch.empty((2, rest_in.shape[1]), dtype=torch.float32, device=rest_in.device).unbind(0)
    check(lib().rg_softmax_merge_dev(_ptr(rest_in), _ptr(own_in), rest_in.shape[0], rest_in.shape[1], _ptr(targets_t),
                                     _ptr(lse), _ptr(loss), _device(rest_in), _stream(rest_in)))
    return lse, loss


def softmax_grad_dev(base_t, queries_t, targets_t, scale, lse, loss, weights, rest=None, mean=None, id_base=0, want_dq=True, want_db=True):
    """rg_softmax_grad_dev: (this shard's part of dq, the shard's rows of db).  lse, loss: over the whole base; rest, mean: this shard's
    (for dq only); weights = dL/dloss [nq]."""
    import torch
    queries_t, base_t, id_base = _rows(queries_t, "queries"), _rows(base_t, "base"), _id_base(id_base)
    _check_pair(queries_t, base_t)
    nq, nb, dim = queries_t.shape[0], base_t.shape[0], base_t.shape[1]
    targets_t = _targets(targets_t, nq, base_t)
    lse, loss, weights = (_check_vector(t, nq, torch.float32, base_t, name) for t, name in ((lse, "lse"), (loss, "loss"), (weights, "weights")))
    if want_dq:
        if rest is None or mean is None or mean.shape != (nq, dim) or mean.dtype != torch.float32 or mean.device != base_t.device or not mean.is_contiguous():
            raise ValueError("rest and mean: the results of softmax_shard_dev(..., want_mean=True) are wanted")
        rest = _check_vector(rest, nq, torch.float32, base_t, "rest")
    dq = torch.empty((nq, dim), dtype=base_t.dtype, device=base_t.device) if want_dq else None
    db = torch.empty((nb, dim), dtype=base_t.dtype, device=base_t.device) if want_db else None
    work, n = _scratch(GRAD, nb if want_db else 0, nq, dim, base_t)
    check(lib().rg_softmax_grad_dev(_ptr(base_t), nb, _stride(base_t), _ptr(queries_t), nq, _stride(queries_t),
                                    dim, _dtype_code(base_t), scale, _ptr(targets_t), id_base,
                                    _ptr(lse), _ptr(loss), _ptr(rest), _ptr(mean), _ptr(weights), _ptr(dq), dim, _ptr(db), dim,
                                    _ptr(work), n, _device(base_t), _stream(base_t)))
    return dq, db


_function = None


def _softmax_function():
    global _function
    if _function is None:
        import torch

        # the calls of softmax_shard_dev and softmax_grad_dev with fewer tensors between them: rest, own, lse and the mean rows in one
        class SoftmaxLoss(torch.autograd.Function):
            @staticmethod
            def forward(ctx, queries, base, targets, scale, want_mean):
                q, b = _rows(queries, "queries"), _rows(base, "base")
                _check_pair(q, b)
                (nq, dim), nb, code = q.shape, b.shape[0], _dtype_code(b)
                loss = b.new_empty(nq, dtype=torch.float32)
                kept = b.new_empty((3 + dim if want_mean else 3) * nq, dtype=torch.float32)
                work, n = _scratch(MEAN if want_mean else STATS, nb, nq, dim, b)
                at = kept.data_ptr()
                check(lib().rg_softmax_shard_dev(b.data_ptr(), nb, _stride(b), q.data_ptr(), nq, _stride(q), dim, code, scale, targets.data_ptr(), 0, at, at + 4 * nq, at + 8 * nq,
                                                 loss.data_ptr(), at + 12 * nq if want_mean else None, work.data_ptr(), n, _device(b), _stream(b)))
                ctx.save_for_backward(queries, base, targets, loss, kept)
                ctx.scale = scale
                return loss

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, weights):
                queries, base, targets, loss, kept = ctx.saved_tensors
                q, b = _rows(queries, "queries"), _rows(base, "base")
                (nq, dim), nb, code = q.shape, b.shape[0], _dtype_code(b)
                weights = weights.contiguous()
                dq = b.new_empty((nq, dim)) if ctx.needs_input_grad[0] else None
                db = b.new_empty((nb, dim)) if ctx.needs_input_grad[1] else None
                work, n = _scratch(GRAD, nb if db is not None else 0, nq, dim, b)
                at = kept.data_ptr()
                check(lib().rg_softmax_grad_dev(b.data_ptr(), nb, _stride(b), q.data_ptr(), nq, _stride(q), dim, code, ctx.scale, targets.data_ptr(), 0, at + 8 * nq, loss.data_ptr(),
                                                at, at + 12 * nq if dq is not None else None, weights.data_ptr(), _ptr(dq), dim, _ptr(db), dim, work.data_ptr(), n, _device(b), _stream(b)))
                return dq, db, None, None, None

        _function = SoftmaxLoss
    return _function


def softmax_loss(queries, base, targets, scale=1.0):
    """Cross entropy of softmax(scale * queries @ base.T) against `targets`, per query [nq] fp32; differentiable (once) in queries and base.

    scale is a number (one held in a GPU tensor is read back, which waits for the GPU).  A learned one goes into the queries, softmax_loss(queries * s, base,
    targets), which gives it its gradient; a scale that requires grad is refused."""
    import torch
    if isinstance(scale, torch.Tensor) and scale.requires_grad and torch.is_grad_enabled():
        raise TypeError("softmax_loss: the scale gets no gradient here; multiply the queries by it instead: softmax_loss(queries * scale, base, targets)")
    targets = _targets(targets, queries.shape[0], base)
    # (the mean rows are for the queries' gradient only; inside forward a leaf wants one even under no_grad)
    return _softmax_function().apply(queries, base, targets, float(scale), queries.requires_grad and torch.is_grad_enabled())
