"""The catalogue head: the softmax cross entropy over the WHOLE item table with its gradients, and scores from tables held in
8 bits, on the HIP kernels of csrc/xent.hip and csrc/int8.hip.

    r = softmax_xent(rows, table, target, scale=10.)       # r.loss, r.lse, r.d_rows, r.d_table (r.d_bias)
    served = quantize_rows(table)                          # once: int8 codes + one fp32 scale per row
    s = int8_scores(user_rows, served)                     # [users, items] scores, rows quantised on the way in

All calls are asynchronous on torch's current stream of the tensors' device and allocate what they return (and their workspace)
there; nothing is kept between calls.  Arguments are checked before anything is launched: a wrong device, type, shape or layout
raises ValueError / TypeError.  Values on the device are not read by the host: what an id out of range or a NaN does is said below.
No reference counterpart: its losses sample their negatives (utils/objectives.py:35-220)."""
import collections
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # nncf_dtype
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}                      # nncf_reduction

XentResult = collections.namedtuple("XentResult", "loss lse d_rows d_table d_bias")


def _matrix(t, name, dtypes):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a tensor on the GPU" % name)
    if t.dtype not in dtypes:
        raise TypeError("%s has dtype %s" % (name, t.dtype))
    if t.dim() != 2:
        raise ValueError("%s must have two dimensions, got shape %s" % (name, tuple(t.shape)))
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("the elements of a row of %s must be adjacent" % name)


def _pitch(t):
    """Elements from row to row; the only row of a matrix has any stride."""
    p = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if p < t.shape[1]:
        raise ValueError("rows overlap (stride %d, width %d)" % (p, t.shape[1]))
    return p


def _vector(t, name, n, dtype, device):
    if t is None and name != "scale":
        return None
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise TypeError("%s must be a tensor on %s" % (name, device))
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError("%s must be a contiguous vector of %d, got shape %s" % (name, n, tuple(t.shape)))
    return t.data_ptr()


def _call(device, fn, *args):
    stream = torch._C._cuda_getCurrentRawStream(device.index)   # current_stream(device).cuda_stream without the object: 0.1 us, not 1.9
    if torch.cuda.current_device() == device.index:
        _lib.check(fn(*args, stream))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, stream))


def softmax_xent(rows, table, target, bias=None, weight=None, scale=1.0, reduction="mean", grad=True):
    """Softmax cross entropy of `rows` [n, d] over every row of `table` [c, d], d <= 128, both float32, float16 or bfloat16:

        z = scale * rows @ table.T + bias;   loss_i = weight_i * (logsumexp(z_i) - z_i[target_i])

    reduction "sum" / "mean" (over the rows that have a target) / "none" (loss [n]; the gradients are those of its sum, so that
    `weight` carries an upstream gradient).  Returns XentResult(loss, lse, d_rows, d_table, d_bias); with grad=False the gradients
    are None.  Loss, lse and d_bias are float32, d_rows / d_table of the inputs' type.  The n x c logits are never stored.

    target (int32): a negative one takes the row out (loss 0, lse 0, gradient 0, whatever its values); one >= c makes the loss and
    the gradients NaN.  bias [c] float32: -inf leaves an item out (its row is not used); a row whose target is left out has loss
    +inf and no gradient.  weight [n] float32: any finite value (a row that is not finite reaches the table's gradient at weight 0 too).
    fp32 magnitudes: include/nncf_hip.h."""
    _matrix(rows, "rows", _DTYPES)
    _matrix(table, "table", _DTYPES)
    n, d = rows.shape
    c = table.shape[0]
    device, dtype = rows.device, rows.dtype
    if table.device != device or table.dtype != dtype:
        raise TypeError("rows and table differ: %s on %s, %s on %s" % (dtype, device, table.dtype, table.device))
    if table.shape[1] != d:
        raise ValueError("rows are %d wide, the table %d" % (d, table.shape[1]))
    if n == 0 or c == 0:
        raise ValueError("no %s" % ("rows" if n == 0 else "items"))
    if target is None:
        raise TypeError("target must be given")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction %r unknown" % (reduction,))
    L = _lib.lib()
    x = _lib.Xent()
    x.rows, x.table = rows.data_ptr(), table.data_ptr()
    x.target = _vector(target, "target", n, torch.int32, device)
    x.bias = _vector(bias, "bias", c, torch.float32, device)
    x.weight = _vector(weight, "weight", n, torch.float32, device)
    x.n, x.c, x.dim, x.dtype, x.reduction, x.scale = n, c, d, _DTYPES[dtype], _REDUCTIONS[reduction], scale
    x.rows_stride, x.table_stride = _pitch(rows), _pitch(table)
    ws_bytes = L.nncf_softmax_xent_ws_bytes(n, c, d, x.dtype, int(bool(grad)))
    if ws_bytes < 0:
        _lib.check(-1)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    loss = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=device)
    lse = torch.empty(n, dtype=torch.float32, device=device)
    x.loss, x.lse = loss.data_ptr(), lse.data_ptr()
    d_rows = d_table = d_bias = None
    if grad:
        d_rows = torch.empty((n, d), dtype=dtype, device=device)
        d_table = torch.empty((c, d), dtype=dtype, device=device)
        x.d_rows, x.d_table = d_rows.data_ptr(), d_table.data_ptr()
        if bias is not None:
            d_bias = torch.empty(c, dtype=torch.float32, device=device)
            x.d_bias = d_bias.data_ptr()
    _call(device, L.nncf_softmax_xent, ctypes.byref(x), ws.data_ptr(), ws_bytes)
    return XentResult(loss, lse, d_rows, d_table, d_bias)


class Int8Rows(object):
    """Rows in 8 bits: `codes` int8 [n, pitch] (-127 .. 127, zeros behind the k-th column) and `scale` float32 [n]; row i stands for
    codes[i, :k] * scale[i].  Made by quantize_rows, or from codes and scales kept elsewhere (pitch = nncf_int8_pitch(k): 64 up to
    k = 64, else the next multiple of 128): those are read once here, which waits for the device and is refused while a graph is captured."""

    __slots__ = ("codes", "scale", "k")

    def __init__(self, codes, scale, k):
        _matrix(codes, "codes", (torch.int8,))
        if codes.shape[1] != _lib.lib().nncf_int8_pitch(k) or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("codes of rows %d wide must be [n, %d], contiguous and 16-byte aligned" % (k, _lib.lib().nncf_int8_pitch(k)))
        _vector(scale, "scale", codes.shape[0], torch.float32, codes.device)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("codes made elsewhere are read when they are taken over: do that before the capture")
        # the products rely on both: sums of 127^2 k stay below 2^31, and columns behind the k-th are multiplied like the others
        for i in range(0, codes.shape[0], 1 << 22):
            part = codes[i:i + (1 << 22)]
            if part[:, :k].amin() < -127 or part[:, k:].any():
                raise ValueError("codes are -127 .. 127, and zeros behind the first %d columns" % k)
        self.codes, self.scale, self.k = codes, scale, k

    @classmethod
    def _of(cls, codes, scale, k):
        self = cls.__new__(cls)
        self.codes, self.scale, self.k = codes, scale, k
        return self

    def __len__(self):
        return self.codes.shape[0]

    def dequantize(self, dtype=torch.float32):
        """The values the codes stand for, [n, k]."""
        if dtype not in _DTYPES:
            raise TypeError("dtype %s" % (dtype,))
        out = torch.empty((len(self), self.k), dtype=dtype, device=self.codes.device)
        _call(out.device, _lib.lib().nncf_dequantize_rows, self.codes.data_ptr(), self.scale.data_ptr(),
              len(self), self.k, out.data_ptr(), _DTYPES[dtype])
        return out


def quantize_rows(x, normalize=False):
    """Rows of `x` [n, k] (float32, float16, bfloat16; k <= 131072) to Int8Rows: code = rint(x * (127 / max |x|)), scale = max |x| / 127
    per row, in fp32.  normalize: the rows stand for their L2-normalised selves (model_framework.py:62-63).  A row with an infinity or
    NaN has scale NaN: so has every score of it."""
    _matrix(x, "x", _DTYPES)
    n, k = x.shape
    L = _lib.lib()
    pitch = L.nncf_int8_pitch(k)
    if pitch < 0:
        raise ValueError("rows of %d columns (1 .. 131072)" % k)
    codes = torch.empty((n, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(n, dtype=torch.float32, device=x.device)
    _call(x.device, L.nncf_quantize_rows, x.data_ptr(), _pitch(x), _DTYPES[x.dtype], n, k, int(bool(normalize)),
          codes.data_ptr(), scale.data_ptr())
    return Int8Rows._of(codes, scale, k)


def int8_scores(rows, table, row_bias=None, col_bias=None, out=None, dtype=torch.float32):
    """Scores of `rows` (Int8Rows, or float rows [m, k] that are quantised first) against `table` (Int8Rows [c, k]):

        out[i, j] = rows.scale_i * table.scale_j * sum_k rows.codes_ik * table.codes_jk + row_bias_i + col_bias_j

    with the integer sum exact.  Biases are float32 vectors.  out: [m, c] of float32, float16 or bfloat16, adjacent columns, any row
    stride (or a new tensor of `dtype`)."""
    if not isinstance(table, Int8Rows):
        raise TypeError("table must be Int8Rows (quantize_rows)")
    L = _lib.lib()
    c, k = len(table), table.k
    device = table.codes.device
    coded = isinstance(rows, Int8Rows)
    if not coded:
        _matrix(rows, "rows", _DTYPES)
        if rows.shape[1] == k and not L.nncf_int8_scores_fused(rows.shape[0], k):
            rows, coded = quantize_rows(rows), True
    m, width, where = (len(rows), rows.k, rows.codes.device) if coded else (rows.shape[0], rows.shape[1], rows.device)
    if width != k:
        raise ValueError("rows are %d wide, the table %d" % (width, k))
    if where != device:
        raise TypeError("rows are on %s, the table on %s" % (where, device))
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError("dtype %s" % (dtype,))
        out = torch.empty((m, c), dtype=dtype, device=device)
    else:
        _matrix(out, "out", _DTYPES)
        if out.device != device or tuple(out.shape) != (m, c):
            raise ValueError("out must be [%d, %d] on %s" % (m, c, device))
    rest = (table.codes.data_ptr(), table.scale.data_ptr(), c, k, _vector(row_bias, "row_bias", m, torch.float32, device),
            _vector(col_bias, "col_bias", c, torch.float32, device), out.data_ptr(), _pitch(out), _DTYPES[out.dtype])
    if coded:
        _call(device, L.nncf_int8_scores, rows.codes.data_ptr(), rows.scale.data_ptr(), m, *rest)
    else:
        _call(device, L.nncf_int8_scores_rows, rows.data_ptr(), _pitch(rows), _DTYPES[rows.dtype], m, *rest)
    return out
