"""The categorical readout on torch CUDA tensors: a layer of 8-bit weights that makes logits, the rules of a generation step,
the draw of a category, and the distillation loss with its gradient (thrml_linear_i8, thrml_adjust_logits,
thrml_draw_categories, thrml_distill_* of include/thrml_b200.h).

A row is one sequence or chain.  Every call runs on the tensors' own device and on that device's current torch stream,
returns before the GPU is done, and can be captured into a CUDA graph once a call has been made on the device before.
Arguments that do not fit raise ThrmlError.  Gradients are returned, as by `estimate_kl_grad`; nothing here is recorded by
autograd.
"""
import ctypes as C

from . import _ffi
from . import engine as _eng
from ._ffi import ThrmlError, lib

torch = None  # imported by the first call: the rest of the package works on host arrays and does without it
_TYPES = {}
_FLOATS, _WHOLE = (0, 1, 2), (3, 4)


def _refuse(why):
    raise ThrmlError(-1, why)


def _load():
    global torch
    if torch is None:
        import torch as module
        _TYPES.update({module.float32: 0, module.bfloat16: 1, module.float16: 2, module.int32: 3, module.int64: 4})
        torch = module


def _device(x, name):
    """The first argument's device: (context handle, stream, device)."""
    if torch is None:
        _load()
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _refuse(f"{name} has to be a CUDA tensor")
    index = x.device.index
    ctx = _eng._default_ctx.get(index)
    if ctx is None:
        if torch.cuda.is_current_stream_capturing():
            _refuse("the first call on a device makes its context, which a stream capture cannot hold: make one call before the capture")
        with torch.cuda.device(index):  # making a context changes the current device
            ctx = _eng.default_context(index)
    return ctx.h, torch.cuda.current_stream(index).cuda_stream, x.device


def _rows(x, name, device, kinds=_FLOATS, rows=None, cols=None):
    """Checks a matrix whose rows are contiguous; (type, pitch)."""
    if not isinstance(x, torch.Tensor) or x.device != device:
        _refuse(f"{name} has to be a tensor on {device}")
    kind = _TYPES.get(x.dtype)
    if kind not in kinds:
        _refuse(f"{name}: {x.dtype} is not taken here")
    if x.dim() != 2 or (rows is not None and x.shape[0] != rows) or (cols is not None and x.shape[1] != cols):
        _refuse(f"{name} has the shape {tuple(x.shape)}, not ({'rows' if rows is None else rows}, {'columns' if cols is None else cols})")
    if x.shape[1] > 1 and x.stride(1) != 1:
        _refuse(f"{name}: the elements of a row have to be contiguous")
    pitch = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    if pitch < x.shape[1]:
        _refuse(f"{name}: rows must not overlap")
    return kind, pitch


def _vector(x, name, device, dtype, n):
    """Pointer of a contiguous vector of n elements, None for None."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.device != device or x.dtype != dtype:
        _refuse(f"{name} has to be a {dtype} tensor on {device}")
    if x.dim() != 1 or (n is not None and x.shape[0] != n) or not x.is_contiguous():
        _refuse(f"{name} has to be a contiguous vector" + ("" if n is None else f" of {n} elements"))
    return x.data_ptr()


def _check(rc):
    if rc:
        _ffi.check(rc)


def _new_or(out, name, like_rows, cols, dtype, device):
    """`out` checked, or a new matrix; (matrix, type, pitch)."""
    if out is None:
        return torch.empty((like_rows, cols), dtype=dtype, device=device), _TYPES[dtype], cols
    kind, pitch = _rows(out, name, device, (_TYPES[dtype],), like_rows, cols)
    return out, kind, pitch


def _workspace8(rows, cols, device):
    """8-bit rows that start on 16-byte boundaries."""
    return torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)


def align_rows_int8(weight):
    """8-bit rows laid out as the product wants them (each on a 16-byte boundary): a view of a padded copy, or `weight` itself
    when it is laid out so already.  Done once, when weights are loaded."""
    _load()
    if not isinstance(weight, torch.Tensor) or weight.dtype != torch.int8 or weight.dim() != 2:
        _refuse("weight has to be an int8 matrix")
    if weight.stride(1) == 1 and weight.stride(0) % 16 == 0 and weight.stride(0) >= weight.shape[1] and weight.data_ptr() % 16 == 0:
        return weight
    out = _workspace8(*weight.shape, weight.device)
    out[:, weight.shape[1]:] = 0
    out = out[:, :weight.shape[1]]
    out.copy_(weight)
    return out


def quantize_rows(x):
    """(q, scale): each row of x in 8 bits with one scale, scale = max |x| / 127 and q = x / scale rounded to nearest even.
    Quantises activations by token and a layer's weights `[channels, inputs]` by channel; q's rows are laid out as the
    product wants them.  A row with an infinity or a NaN gets a scale that makes NaN of everything computed from it."""
    h, stream, dev = _device(x, "x")
    kind, pitch = _rows(x, "x", dev)
    rows, cols = x.shape
    q, scale = _workspace8(rows, cols, dev), torch.empty(rows, dtype=torch.float32, device=dev)
    _check(lib().thrml_quantize_rows_i8(h, stream, rows, cols, x.data_ptr(), kind, pitch, q.data_ptr(), q.shape[1], scale.data_ptr()))
    return q[:, :cols], scale


def _weight8(weight, weight_scale, bias, device, cols):
    if not isinstance(weight, torch.Tensor) or weight.device != device or weight.dtype != torch.int8 or weight.dim() != 2 or weight.shape[1] != cols:
        _refuse(f"weight has to be an int8 matrix [channels, {cols}] on {device}")
    if cols > 1 and weight.stride(1) != 1:
        _refuse("weight: the elements of a row have to be contiguous")
    n = weight.shape[0]
    pitch = weight.stride(0) if n > 1 else (cols + 15) // 16 * 16
    return n, pitch, _vector(weight_scale, "weight_scale", device, torch.float32, n), _vector(bias, "bias", device, torch.float32, n)


def int8_matmul(q, q_scale, weight, weight_scale, bias=None, out_dtype=None, out=None):
    """(q @ weight.T) * q_scale[:, None] * weight_scale + bias: 8-bit rows `q [tokens, inputs]` and `weight [channels, inputs]`
    (int8, rows on 16-byte boundaries: see `align_rows_int8`), one f32 scale per token and channel, f32 bias.  The sums are
    exact; the result is rounded once to `out_dtype` (float32, bfloat16 or float16; float32 by default)."""
    h, stream, dev = _device(q, "q")
    if q.dtype != torch.int8 or q.dim() != 2 or (q.shape[1] > 1 and q.stride(1) != 1):
        _refuse("q has to be an int8 matrix with contiguous rows")
    m, k = q.shape
    pitch = q.stride(0) if m > 1 else (k + 15) // 16 * 16
    scale = _vector(q_scale, "q_scale", dev, torch.float32, m)
    n, w_pitch, w_scale, b = _weight8(weight, weight_scale, bias, dev, k)
    if scale is None or w_scale is None:
        _refuse("q_scale and weight_scale are needed")
    if out_dtype is None:
        out_dtype = torch.float32 if out is None else out.dtype
    if _TYPES.get(out_dtype) not in _FLOATS:
        _refuse(f"out_dtype: {out_dtype} is not taken here")
    out, out_kind, out_pitch = _new_or(out, "out", m, n, out_dtype, dev)
    _check(lib().thrml_matmul_i8(h, stream, m, n, k, q.data_ptr(), pitch, scale, weight.data_ptr(), w_pitch, w_scale, b, out.data_ptr(), out_kind, out_pitch))
    return out


def int8_linear(x, weight, weight_scale, bias=None, out_dtype=None, out=None):
    """x @ W.T + bias with W = weight * weight_scale[:, None] in 8 bits: `quantize_rows(x)` and `int8_matmul` in one call.  The
    result has x's type unless `out_dtype` says otherwise."""
    h, stream, dev = _device(x, "x")
    kind, pitch = _rows(x, "x", dev)
    m, k = x.shape
    n, w_pitch, w_scale, b = _weight8(weight, weight_scale, bias, dev, k)
    if w_scale is None:
        _refuse("weight_scale is needed")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    if _TYPES.get(out_dtype) not in _FLOATS:
        _refuse(f"out_dtype: {out_dtype} is not taken here")
    out, out_kind, out_pitch = _new_or(out, "out", m, n, out_dtype, dev)
    q_pitch = (k + 15) // 16 * 16
    space = torch.empty(m * q_pitch + 4 * m, dtype=torch.int8, device=dev)  # the rows in 8 bits, then their scales
    at = space.data_ptr()
    _check(lib().thrml_linear_i8(h, stream, m, n, k, x.data_ptr(), kind, pitch, at, q_pitch, at + m * q_pitch, weight.data_ptr(), w_pitch, w_scale, b, out.data_ptr(),
                                 out_kind, out_pitch))
    return out


def adjust_logits(logits, *, history=None, history_ptr=None, n_prompt=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, bias_ptr=None,
                  mask=None, mask_rows=None, out=None):
    """The rules of one generation step on `logits [rows, categories]`, in this order:

    penalties  for what the row has seen: tokens history[history_ptr[r]:history_ptr[r + 1]] (int32 or int64; history_ptr int64),
               the first n_prompt[r] (int32) being its prompt.  Seen at all: x / repetition where x > 0, else x * repetition; seen
               o > 0 times behind the prompt: x - frequency * o - presence.  One f32 value per row each.
    biases     x + bias_values (f32) for the entries bias_ptr[r]:bias_ptr[r + 1] (int64) with bias_ids (int32) equal to the category;
               entries that repeat a category stand next to each other and add up.
    mask       -inf where bit k & 31 of word k >> 5 of the row's mask is 0; mask int32 [masks, words], mask_rows (int32) says
               which mask a row has, -1 = none; without mask_rows, row r has mask r.

    Ids outside the categories are padding.  `out` may be `logits` itself."""
    h, stream, dev = _device(logits, "logits")
    kind, pitch = _rows(logits, "logits", dev)
    rows, cols = logits.shape
    if out is not logits:
        out, _, out_pitch = _new_or(out, "out", rows, cols, logits.dtype, dev)
    else:
        out_pitch = pitch
    r = _ffi.LogitRules()
    f32 = torch.float32
    if history is not None:
        if not isinstance(history, torch.Tensor) or _TYPES.get(history.dtype) not in _WHOLE:
            _refuse("history has to be an int32 or int64 tensor")
        r.history_type = _TYPES[history.dtype]
        r.history = _vector(history, "history", dev, history.dtype, None) or None
        r.history_ptr = _vector(history_ptr, "history_ptr", dev, torch.int64, rows + 1)
        if history_ptr is None:
            _refuse("history needs history_ptr")
        r.n_prompt = _vector(n_prompt, "n_prompt", dev, torch.int32, rows)
        r.repetition = _vector(repetition, "repetition", dev, f32, rows)
        r.frequency = _vector(frequency, "frequency", dev, f32, rows)
        r.presence = _vector(presence, "presence", dev, f32, rows)
    elif not (history_ptr is n_prompt is repetition is frequency is presence is None):
        _refuse("penalties need a history")
    if bias_ids is not None:
        if bias_values is None or bias_ptr is None:
            _refuse("bias_ids needs bias_values and bias_ptr")
        r.bias_ids = _vector(bias_ids, "bias_ids", dev, torch.int32, None) or None
        r.bias_values = _vector(bias_values, "bias_values", dev, f32, bias_ids.shape[0]) or None
        r.bias_ptr = _vector(bias_ptr, "bias_ptr", dev, torch.int64, rows + 1)
    elif not (bias_values is bias_ptr is None):
        _refuse("bias_values and bias_ptr need bias_ids")
    if mask is not None:
        _, r.mask_pitch = _rows(mask, "mask", dev, (3,))
        r.n_masks = mask.shape[0]
        if mask.shape[1] < (cols + 31) // 32:
            _refuse(f"mask: {mask.shape[1]} words are fewer than {cols} categories need")
        if mask_rows is None and mask.shape[0] != rows:
            _refuse("mask without mask_rows has one mask for each row")
        r.mask = mask.data_ptr()
        r.mask_rows = _vector(mask_rows, "mask_rows", dev, torch.int32, rows)
    elif mask_rows is not None:
        _refuse("mask_rows needs mask")
    _check(lib().thrml_adjust_logits(h, stream, rows, cols, logits.data_ptr(), kind, pitch, out.data_ptr(), out_pitch, C.byref(r)))
    return out


def draw_categories(logits, key, *, beta=None, row_offset=0, noise=None, out=None):
    """One category per row of `logits [rows, categories]` with probability softmax(beta * logits), as int64: the Gumbel-argmax draw
    of the categorical samplers, argmax_k beta * l_k - log(-log(u_k)), ties to the lowest category.  beta: one f32 value per
    row (None = 1); infinity takes the largest logit.  Categories at -inf or NaN are never drawn; a row without any other
    gets -1.

    key: the seed of an RngKey (or the RngKey); row r's noise depends on the key and on row_offset + r alone, so rows may be
    sharded.  noise: uniforms in (0, 1) `[rows, categories]` f32 to use instead."""
    h, stream, dev = _device(logits, "logits")
    kind, pitch = _rows(logits, "logits", dev)
    rows, cols = logits.shape
    u, u_pitch = None, 0
    if noise is not None:
        _, u_pitch = _rows(noise, "noise", dev, (0,), rows, cols)
        u = noise.data_ptr()
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    else:
        _vector(out, "out", dev, torch.int64, rows)
    key = key.seed() if hasattr(key, "seed") else int(key)
    if not 0 <= key < 1 << 64:
        _refuse("key is not a 64-bit number")
    _check(lib().thrml_draw_categories(h, stream, rows, cols, logits.data_ptr(), kind, pitch, _vector(beta, "beta", dev, torch.float32, rows), key, int(row_offset), u, u_pitch,
                                       out.data_ptr()))
    return out


def _distill_args(logits, ids, teacher, beta, weight):
    h, stream, dev = _device(logits, "logits")
    kind, pitch = _rows(logits, "logits", dev)
    rows, cols = logits.shape
    ids_kind, ids_pitch = _rows(ids, "ids", dev, _WHOLE, rows)
    top = ids.shape[1]
    t_kind, t_pitch = _rows(teacher, "teacher", dev, _FLOATS, rows, top)
    return (h, stream, rows, cols, logits.data_ptr(), kind, pitch, top, ids.data_ptr(), ids_kind, ids_pitch, teacher.data_ptr(), t_kind, t_pitch, float(beta),
            _vector(weight, "weight", dev, torch.float32, rows))


def distill_loss(logits, ids, teacher, *, beta=1.0, weight=None):
    """(loss, lse) of a student's `logits [rows, categories]` against a teacher's top logits: `teacher [rows, top]` at the categories
    `ids [rows, top]` (int32 or int64; ids outside the categories, or teacher logits of -inf, are not listed; top <= 1024).

    loss[r] = sum_j p_j (log p_j - log q_id(j)) with p = softmax over the listed of beta * teacher and q = softmax of beta * logits;
    lse = logsumexp(beta * logits), for `distill_grad`.  Rows whose weight is 0 are padding: they are not read and have loss 0."""
    a = _distill_args(logits, ids, teacher, beta, weight)
    loss = torch.empty((2, logits.shape[0]), dtype=torch.float32, device=logits.device)
    _check(lib().thrml_distill_loss(*a, loss.data_ptr(), loss.data_ptr() + 4 * logits.shape[0]))
    return loss[0], loss[1]


def distill_grad(logits, lse, ids, teacher, *, beta=1.0, weight=None, out=None):
    """The gradient of sum_r weight[r] * loss[r] by the logits, in their type, from `distill_loss`'s lse: weight (f32 per row, None = 1)
    is what comes from above."""
    a = _distill_args(logits, ids, teacher, beta, weight)
    out, _, pitch = _new_or(out, "out", *logits.shape, logits.dtype, logits.device)
    lse_ptr = _vector(lse, "lse", logits.device, torch.float32, logits.shape[0])
    _check(lib().thrml_distill_grad(*a, lse_ptr, out.data_ptr(), pitch))
    return out


def distill_step(logits, ids, teacher, *, beta=1.0, weight=None, out=None):
    """(loss, gradient) in one call: `distill_loss` and `distill_grad` for weights that are known beforehand.  `out`: the
    gradient."""
    a = _distill_args(logits, ids, teacher, beta, weight)
    out, _, pitch = _new_or(out, "out", *logits.shape, logits.dtype, logits.device)
    loss = torch.empty((2, logits.shape[0]), dtype=torch.float32, device=logits.device)  # and lse
    _check(lib().thrml_distill_step(*a, loss.data_ptr(), loss.data_ptr() + 4 * logits.shape[0], out.data_ptr(), pitch))
    return loss[0], out
