"""Points held in 8 bits, the product of rows with them and its gradient, and the teacher's loss, on torch tensors.

Beside the graph and the embedding (no counterpart in the reference): a bank of points in a quarter of f32's memory, an encoder trained so that the
softmax of its scores against the bank follows the graph's edge probabilities.

    bank = Points8(capacity=n, dim=784)
    bank.write(x)                                          # quantised as it is written
    graph = KGraph.bruteforce_l2_points8(bank, 12)         # the exact graph of the points as held
    logits = bank.product(q, dtype=torch.bfloat16)         # [m, n]
    loss, stats, dlogits = teacher_loss(logits, idx, proba, grad=True)
    dq = bank.product_grad(dlogits)                        # [m, dim]

Tensors live on one GPU; the work goes to torch's current stream of that GPU and the calls return at once: they neither synchronise nor
allocate outside torch's allocator, so they can be captured into a graph (which keeps neither the store nor the caller's tensors alive).  Results are
detached: gradients are the calls product_grad and teacher_loss / teacher_grad.  A tensor of the caller's that a call writes to counts as changed in
place, and so do codes() and scales() at every write.  The formats, formulas and edge cases are those of ae_points8_* and ae_teacher_* in include/annembed_hip.h.
"""
import ctypes as C
import functools

import torch

from . import _lib as L
from ._lib import AnnembedError, check

_TYPES = {torch.float32: L.AE_TYPE_F32, torch.bfloat16: L.AE_TYPE_BF16, torch.float16: L.AE_TYPE_F16}
_KINDS = {"proba": L.AE_TEACHER_PROBA, "logits": L.AE_TEACHER_LOGITS}


def _bad(msg):
    return AnnembedError(L.AE_ERR_INVALID_ARG, msg)


def _rows(t, what, device, shape=None):
    """pointer, type and row stride of a 2-D tensor whose rows are contiguous"""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise _bad("%s has to be a 2-D tensor" % what)
    kind, (rows, cols), (ld, inner) = _TYPES.get(t.dtype), t.shape, t.stride()
    if kind is None:
        raise _bad("%s is %s: float32, bfloat16 and float16 are taken" % (what, t.dtype))
    if t.device != device:
        raise _bad("%s is on %s, not on %s" % (what, t.device, device))
    if shape is not None and (rows, cols) != shape:
        raise _bad("%s has shape %s, not %s" % (what, (rows, cols), shape))
    if inner != 1 and cols > 1:
        raise _bad("%s: the elements of a row have to be next to each other (stride %d)" % (what, inner))
    if ld < cols:
        if rows > 1:
            raise _bad("%s: rows that overlap (stride %d of %d elements)" % (what, ld, cols))
        ld = cols
    return t.data_ptr(), kind, ld


def _vector(t, what, device, n, dtypes):
    """pointer of a contiguous 1-D tensor of n elements, or None"""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.shape != (n,):
        raise _bad("%s has to be a 1-D tensor of %d elements of %s" % (what, n, " or ".join(str(d) for d in dtypes)))
    if t.device != device:
        raise _bad("%s is on %s, not on %s" % (what, t.device, device))
    if n > 1 and t.stride(0) != 1:
        raise _bad("%s has to be contiguous" % what)
    return t.data_ptr()


_INDEX = (torch.int32, torch.uint32)


# the current stream of a device as an integer: the public torch.cuda.current_stream() builds an object first, for 2.5 us a call
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device   # (the public one looks whether CUDA is initialised first)


def _call(device, fn, *args):
    """the library call on torch's current stream of `device`, which has to be the current device while it runs"""
    f, index = getattr(L.load(), fn), device.index
    if _device() == index:
        rc = f(*args, _stream(index))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _stream(index))
    if rc != L.AE_OK:   # (none of these calls leaves a warning)
        check(rc)


@functools.lru_cache(maxsize=1024)
def _loss_work(rows, cols):
    """bytes of scratch, asked for once for each size"""
    need = C.c_uint64()
    check(L.load().ae_teacher_loss_work(rows, cols, C.byref(need)))
    return need.value


# what is written behind torch's back has another version, so that autograd refuses to go back through what it held before
_changed = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version   # (of a list; the public one looks at it first)


class _Store:
    """the handle, and the bytes of scratch of its calls, asked for once for each size; views of its memory keep it alive"""

    def __init__(self, h):
        def asked(fn):
            @functools.lru_cache(maxsize=1024)
            def need(*sizes):
                bytes_ = C.c_uint64()
                check(fn(h, *sizes, C.byref(bytes_)))
                return bytes_.value
            return need

        self.h = h
        self.product_work, self.product_grad_work = asked(L.load().ae_points8_product_work), asked(L.load().ae_points8_product_grad_work)

    def __del__(self):
        try:
            L.load().ae_points8_destroy(self.h)
        except Exception:
            pass


class _View:
    def __init__(self, store, ptr, shape, strides):
        self.store = store
        self.__cuda_array_interface__ = {"shape": shape, "strides": strides, "typestr": "|u1", "data": (ptr, False), "version": 2}


class Points8:
    """Room for `capacity` points of `dim` coordinates in 8 bits: e4m3 codes with a power-of-two scale for each block of 128 coordinates."""

    def __init__(self, capacity, dim, device=None):
        if not 0 < int(capacity) < 0xFFFFFFFF or not 0 < int(dim) <= 1 << 20:
            raise _bad("Points8: %s points of %s coordinates are out of range" % (capacity, dim))
        if not torch.cuda.is_available():
            raise AnnembedError(L.AE_ERR_NO_DEVICE, "no HIP device available (annembed_amd is GPU-only)")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise _bad("Points8: %s is no GPU" % device)
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        self.capacity, self.dim = int(capacity), int(dim)
        h, row_bytes, stride, codes, scales = C.c_void_p(), C.c_uint64(), C.c_uint64(), C.c_void_p(), C.c_void_p()
        with torch.cuda.device(self.device):
            check(L.load().ae_points8_create(self.capacity, self.dim, C.byref(h)))
            self._store = _Store(h)
            check(L.load().ae_points8_info(h, None, None, C.byref(row_bytes), C.byref(stride)))
            check(L.load().ae_points8_device(h, C.byref(codes), C.byref(scales)))
            blocks = -(-self.dim // 128)
            c = torch.as_tensor(_View(self._store, codes.value, (self.capacity, self.dim), (row_bytes.value, 1)), device=self.device)
            self._codes = c.view(torch.float8_e4m3fn)
            self._scales = torch.as_tensor(_View(self._store, scales.value, (self.capacity, blocks), (1, stride.value)), device=self.device)
            self._views = [self._codes, self._scales]

    @property
    def handle(self):
        return self._store.h

    def codes(self):
        """the codes themselves, [capacity, dim] float8_e4m3fn: the store's own memory"""
        return self._codes

    def scales(self):
        """the scale bytes, [capacity, ceil(dim / 128)] uint8: a block's values are code * 2^(byte - 127)"""
        return self._scales

    def _range(self, n, first):
        first = int(first)
        n = self.capacity - first if n is None else int(n)
        if first < 0 or n < 0 or first + n > self.capacity:
            raise _bad("points %d ... + %d are outside a store of %d" % (first, n, self.capacity))
        return n, first

    def write(self, x, first=0, slots=None):
        """rows of x into the points first, first + 1, ... or into `slots` (int32; -1 is skipped, the last of equal slots is held)"""
        p, ty, ld = _rows(x, "x", self.device)
        n = x.shape[0]
        if x.shape[1] != self.dim:
            raise _bad("x has %d coordinates, the store %d" % (x.shape[1], self.dim))
        s = _vector(slots, "slots", self.device, n, _INDEX)
        n, first = (n, 0) if slots is not None else self._range(n, first)
        _call(self.device, "ae_points8_write", self._store.h, p, ty, n, ld, first, s if n else None)
        _changed(self._views)

    def read(self, n=None, first=0, slots=None, dtype=torch.float32, out=None):
        """the values held in points first ... first + n - 1, or in `slots` (-1 reads as zeros, others outside the store as NaN)"""
        if slots is not None:
            many = slots.numel() if isinstance(slots, torch.Tensor) else 0
            if n is not None and n != many:
                raise _bad("%s points from %d slots" % (n, many))
            n, first = many, 0
        else:
            n, first = self._range(n, first)
        s = _vector(slots, "slots", self.device, n, _INDEX)
        given = out is not None
        if not given:
            out = torch.empty(n, self.dim, dtype=dtype, device=self.device)
        p, ty, ld = _rows(out, "out", self.device, (n, self.dim))
        _call(self.device, "ae_points8_read", self._store.h, first, s if n else None, n, p, ty, ld)
        if given:
            _changed([out])
        return out

    def _work(self, work, need):
        if work is None:
            work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        elif not isinstance(work, torch.Tensor) or work.device != self.device or not work.is_contiguous():
            raise _bad("work has to be a contiguous tensor on %s" % self.device)
        return (None, 0, None) if work is None else (work.data_ptr(), work.numel() * work.element_size(), work)

    def product(self, x, n=None, first=0, dtype=torch.float32, out=None, work=None, x_first=0, m=None):
        """<x_i, p_j> for the rows of x -- quantised as write() would -- or for m points of another store, and points first ... first + n - 1"""
        n, first = self._range(n, first)
        if isinstance(x, Points8):
            m, x_first = x._range(m, x_first)
        else:
            xp, xt, xl = _rows(x, "x", self.device)
            if x_first != 0 or m not in (None, x.shape[0]):
                raise _bad("x_first and m choose points of another store: of a tensor all %d rows are taken" % x.shape[0])
            m = x.shape[0]
            if x.shape[1] != self.dim:
                raise _bad("x has %d coordinates, the store %d" % (x.shape[1], self.dim))
        given = out is not None
        if not given:
            out = torch.empty(m, n, dtype=dtype, device=self.device)
        p, ty, ld = _rows(out, "out", self.device, (m, n))
        if isinstance(x, Points8):
            _call(self.device, "ae_points8_product_points", self._store.h, first, n, x._store.h, x_first, m, p, ty, ld)
        else:
            wp, wn, keep = self._work(work, self._store.product_work(n, m))
            _call(self.device, "ae_points8_product", self._store.h, first, n, xp, xt, m, xl, p, ty, ld, wp, wn)
        if given:
            _changed([out])
        return out

    def product_grad(self, dc, n=None, first=0, dtype=torch.float32, out=None, work=None):
        """the gradient of product() to its rows from the gradient of its result: sum_j dc[i][j] * p_j"""
        n, first = self._range(n, first)
        dp, dt, dl = _rows(dc, "dc", self.device)
        m = dc.shape[0]
        if dc.shape[1] != n:
            raise _bad("dc has %d columns for %d points" % (dc.shape[1], n))
        given = out is not None
        if not given:
            out = torch.empty(m, self.dim, dtype=dtype, device=self.device)
        p, ty, ld = _rows(out, "out", self.device, (m, self.dim))
        wp, wn, keep = self._work(work, self._store.product_grad_work(n, m, dt))
        _call(self.device, "ae_points8_product_grad", self._store.h, first, n, dp, dt, m, dl, p, ty, ld, wp, wn)
        if given:
            _changed([out])
        return out


def _list(idx, values, rows, device):
    """pointers, length and stride of a teacher's lists [rows, k]"""
    if not isinstance(idx, torch.Tensor) or idx.dim() != 2 or idx.dtype not in _INDEX or idx.shape[0] != rows:
        raise _bad("idx has to be an int32 tensor of %d rows" % rows)
    if not isinstance(values, torch.Tensor) or values.shape != idx.shape or values.dtype != torch.float32:
        raise _bad("the list's values have to be a float32 tensor of idx's shape")
    if idx.device != device or values.device != device:
        raise _bad("the lists are on %s and %s, not on %s" % (idx.device, values.device, device))
    k, (ld, inner), theirs = idx.shape[1], idx.stride(), values.stride()
    if rows <= 1:
        if k > 1 and (inner != 1 or theirs[1] != 1):
            raise _bad("the lists' entries have to be next to each other")
        ld = k
    elif (ld, inner) != theirs or (k > 1 and inner != 1) or ld < k:
        raise _bad("idx and the list's values have to have the same strides, entries next to each other")
    return idx.data_ptr(), values.data_ptr(), k, ld


def _kind(teacher):
    if teacher not in _KINDS:
        raise _bad("teacher has to be 'proba' or 'logits', not %r" % (teacher,))
    return _KINDS[teacher]


def _gpu(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _bad("%s has to be a tensor on a GPU" % what)
    return t.device


_F32 = (torch.float32,)


def teacher_loss(logits, idx, values, teacher="proba", temperature=1.0, row_weight=None, grad=False, work=None):
    """Cross entropy of every row of `logits` against the teacher's list (idx, values), relative to the teacher's own entropy.

    idx [rows, k] int32: columns, -1 for an empty place; values [rows, k] float32: the teacher's probabilities (teacher="proba"; a graph row's
    of NodeParams) or logits (teacher="logits": p = softmax(values / temperature) over the list).  Returns (loss [rows], stats [rows, 2]) or,
    with grad=True or a tensor to write to (`logits` itself is one), (loss, stats, gradient of loss.sum() to the logits in their type)."""
    device = _gpu(logits, "logits")
    p, ty, ld = _rows(logits, "logits", device)
    rows, cols = logits.shape
    ip, vp, k, ldk = _list(idx, values, rows, device)
    wp = _vector(row_weight, "row_weight", device, rows, _F32)
    loss = torch.empty(rows, dtype=torch.float32, device=device)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=device)
    gp, gl, g = None, 0, None
    if grad is not False and grad is not None:
        g = torch.empty(rows, cols, dtype=logits.dtype, device=device) if grad is True else grad
        gp, gt, gl = _rows(g, "grad", device, (rows, cols))
        if gt != ty:
            raise _bad("grad is %s, the logits %s" % (g.dtype, logits.dtype))
    need = _loss_work(rows, cols)
    if work is None:
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    elif not isinstance(work, torch.Tensor) or work.device != device or not work.is_contiguous():
        raise _bad("work has to be a contiguous tensor on %s" % device)
    _call(device, "ae_teacher_loss", p, ty, rows, cols, ld, ip, vp, k, ldk, _kind(teacher), float(temperature), wp, loss.data_ptr(), stats.data_ptr(), gp, gl,
          None if work is None else work.data_ptr(), 0 if work is None else work.numel() * work.element_size())
    if g is not None and grad is not True:
        _changed([g])
    return (loss, stats) if g is None else (loss, stats, g)


def teacher_grad(logits, stats, idx, values, dloss=None, teacher="proba", temperature=1.0, out=None):
    """The gradient to the logits from the statistics that teacher_loss returned for them, under each row's upstream gradient dloss [rows]
    (with the row's weight in it; None: 1).  `out` may be the logits."""
    device = _gpu(logits, "logits")
    p, ty, ld = _rows(logits, "logits", device)
    rows, cols = logits.shape
    ip, vp, k, ldk = _list(idx, values, rows, device)
    if not isinstance(stats, torch.Tensor) or stats.shape != (rows, 2) or stats.dtype != torch.float32 or stats.device != device or not stats.is_contiguous():
        raise _bad("stats has to be the [%d, 2] float32 tensor of teacher_loss" % rows)
    up = _vector(dloss, "dloss", device, rows, _F32)
    g = torch.empty(rows, cols, dtype=logits.dtype, device=device) if out is None else out
    gp, gt, gl = _rows(g, "out", device, (rows, cols))
    if gt != ty:
        raise _bad("out is %s, the logits %s" % (g.dtype, logits.dtype))
    _call(device, "ae_teacher_grad", p, ty, rows, cols, ld, stats.data_ptr(), ip, vp, k, ldk, _kind(teacher), float(temperature), up, gp, gl)
    if out is not None:
        _changed([g])
    return g
