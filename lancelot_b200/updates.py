"""Clients' updates: held as 8-bit integers with scales, formed in 8 bits, bounded.

``UpdateCache`` takes the place of the ``[n_clients][dim]`` tensor of updates in ``EncryptedKrum.round``, ``EncryptedKrum.encrypt_slices``
and ``plaintext_krum``: a quarter of the memory (20 clients of 11 M values: 0.22 GB instead of 0.9), written as updates arrive, with the
error feedback of 8-bit uploads, and read back a range of pages at a time.  ``low_rank_update`` forms an update from 8-bit factors,
``fp8_linear`` trains a client's layer with products in 8-bit floating point, ``flat_updates`` bounds what came of it and lays it out as rows.
The reference keeps every update as a list of doubles (lancelot-main-GPU/utils/byzantine_fl.py:478-490) and has none of these.
"""
import operator

import torch

from .cabi import FP8_TYPES


class UpdateCache:
    """Updates of n_clients clients, dim values each, in pages of ``page`` codes with a scale for every ``group`` of them (a power of two
    from 32 on; 0: one scale a page).  ``lb``: the ``cabi.Context`` whose device holds the cache."""

    def __init__(self, lb, n_clients, dim, page=32768, group=128):
        if n_clients < 1 or dim < 1:
            raise ValueError("a cache holds at least one client and one value")
        if page < 16 or page % 16:
            raise ValueError("a page holds a multiple of 16 codes")
        if group and (group < 32 or group & (group - 1)):
            raise ValueError("group is 0 or a power of two from 32 on")
        self.lb, self.page, self.group = lb, page, group
        self.shape = torch.Size((n_clients, dim))
        self.device = torch.device("cuda", lb.device)
        self.pages = -(-dim // page)
        n = n_clients * self.pages
        self.codes = torch.zeros(n, page, dtype=torch.int8, device=self.device)
        self.scales = torch.zeros(n, -(-page // group) if 0 < group < page else 1, device=self.device)
        self.table = torch.arange(n, dtype=torch.int32, device=self.device).view(n_clients, self.pages)

    def _rows(self, clients):
        """the slots of some clients: all of them (None), one (an integer) or a contiguous range (a slice)"""
        if clients is None:
            return self.table
        if isinstance(clients, slice):
            rows = self.table[clients]
            if not rows.is_contiguous():
                raise ValueError("clients is a contiguous range")
            return rows
        try:
            c = operator.index(clients)
        except TypeError:
            raise ValueError("clients is None, an integer or a contiguous range") from None
        if not 0 <= c < self.shape[0]:
            raise ValueError("client %d is not in the cache" % c)
        return self.table[c:c + 1]

    def write(self, values, clients=None, residual=None, residual_out=None, lengths=None):
        """Quantises updates into the cache: values [dim] of one client or [k][dim] of a range (float32, bfloat16, float16, on the cache's device;
        float64 is rounded to float32).  residual is added first; residual_out (may be residual) gets what the rounding lost, exactly:
        handing it on to the next round's write makes the sum of what was sent follow the sum of the updates."""
        rows = self._rows(clients)
        as_rows = lambda t: t.unsqueeze(0) if t is not None and t.dim() == 1 else t  # noqa: E731
        values = as_rows(values.float() if values.dtype == torch.float64 else values)
        if tuple(values.shape) != (rows.shape[0], self.shape[1]):
            raise ValueError("values must be [%d][%d]" % (rows.shape[0], self.shape[1]))
        self.lb.quantize_rows(values, self.codes, self.scales, group=self.group, slots=rows, lengths=lengths, residual=as_rows(residual),
                              residual_out=as_rows(residual_out))

    def read(self, clients=None, first_page=0, n_pages=None, dtype=torch.float32, out=None):
        """[k][columns] values of some clients: those of n_pages pages from first_page on, up to the end of the update unless ``out`` is wider
        (what lies behind the end reads as zeros)"""
        rows = self._rows(clients)
        n_pages = self.pages - first_page if n_pages is None else n_pages
        if first_page < 0 or n_pages < 0 or first_page + n_pages > self.pages:
            raise ValueError("an update has %d pages" % self.pages)
        cols = min(n_pages * self.page, self.shape[1] - first_page * self.page) if out is None else out.shape[-1]
        if cols > n_pages * self.page or cols <= (n_pages - 1) * self.page:
            raise ValueError("out does not end in the last of the %d pages" % n_pages)
        slots = rows if n_pages == self.pages else rows[:, first_page:first_page + n_pages].contiguous()
        return self.lb.dequantize_rows(self.codes, self.scales, max(cols, 0), group=self.group, slots=slots, n_rows=rows.shape[0], dtype=dtype, out=out)

    def distances(self, clients=None):
        """squared distances between all pairs of updates, [k][k] float64"""
        return self.lb.int8_distances(self.codes, self.scales, self._rows(clients), group=self.group)


def quantize_matrix(lb, x):
    """x [rows][cols] -> (codes [rows][cols] int8, scales [rows]): one scale a row, the form that ``cabi.Context.int8_matmul`` takes.  Rows of
    codes start on 16-byte boundaries whatever cols is."""
    rows, cols = x.shape
    codes = torch.empty(rows, max(16, -(-cols // 16) * 16), dtype=torch.int8, device=x.device)
    scales = (torch.empty if cols else torch.zeros)(rows, 1, device=x.device)  # a row of no columns has no page to be written: scale 0
    lb.quantize_rows(x, codes, scales)
    return codes[:, :cols], scales.view(-1)


def low_rank_update(lb, factors, out=None):
    """The flat float32 update of matrices given by 8-bit factors.  factors: for every matrix W = B A^T a tuple (b [rows][rank], b_scale, a [cols][rank],
    a_scale), either int8 with a scale per row (``quantize_matrix``) or 8-bit floats with scales for blocks of 128
    (``cabi.Context.quantize_fp8``); the matrices follow one another row by row.  Clients' factors cannot be averaged for the update (the
    mean of products is not the product of means), so the product is formed before the encryption."""
    sizes = [b.shape[0] * a.shape[0] for b, _, a, _ in factors]
    if out is None:
        out = torch.empty(sum(sizes), device="cuda:%d" % lb.device)
    if out.dim() != 1 or out.numel() != sum(sizes) or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError("out must be a contiguous float32 vector of %d values" % sum(sizes))
    at = 0
    for (b, b_scale, a, a_scale), size in zip(factors, sizes):
        to = out[at:at + size].view(b.shape[0], a.shape[0])
        if b.dtype in FP8_TYPES:
            lb.fp8_matmul(b, b_scale, a, a_scale, out=to)
        else:
            lb.int8_matmul(b, a, b_scale, a_scale, out=to)
        at += size
    return out


def fp8_linear(lb, x, w, grad_dtype=torch.float8_e4m3fn):
    """y = x w^T with gradients, x [..., k], w [n][k] (float32, bfloat16, float16, on the device of lb): the three products of a training step in
    8-bit floating point.  x is quantised in blocks of 128 values along what a product sums over, w in blocks of 128 x 128; the gradient of y as x,
    to grad_dtype.  y and the gradients have the types of x and of their tensors.  Gradients of y below some 1e-30 lose bits (the products of scales leave the
    normal numbers of 32 bits): a loss that small is scaled up first.  What is kept for the backward pass are the codes.  The gradients
    themselves are not differentiable.  In a graph capture take them with ``torch.autograd.grad``"""
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError("x must be [..., k] and w [n][k]")
    if grad_dtype not in FP8_TYPES:
        raise ValueError("grad_dtype must be float8_e4m3fn or float8_e5m2")
    return lb.fp8_linear(x, w, grad_dtype)


def flat_updates(lb, updates, max_norm=None, out=None, dtype=torch.float32):
    """Clients' updates, for each a list of tensors (the parameters' differences or gradients of its model), as the matrix [n_clients][dim] that
    ``EncryptedKrum.round``, ``plaintext_krum`` and ``UpdateCache.write`` take, scaled down to max_norm where their norm over all tensors is larger
    -> (matrix, norms [n_clients] float64)"""
    if out is None:
        dims = {sum(t.numel() for t in tensors) for tensors in updates}
        if len(dims) > 1:
            raise ValueError("the updates have different numbers of values")
        out = torch.empty(len(updates), dims.pop() if dims else 0, dtype=dtype, device="cuda:%d" % lb.device)
    return out, lb.clip_updates(updates, max_norm, out=out)
