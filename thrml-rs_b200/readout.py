"""The categorical readout on torch CUDA tensors: a layer of 8-bit weights that makes logits, the rules of a generation step,
the draw of a category, and the distillation loss with its gradient (thrml_linear_i8, thrml_adjust_logits,
thrml_draw_categories, thrml_distill_* of include/thrml_b200.h).

A row is one sequence or chain.  Every call runs on the tensors' own device and on that device's current torch stream,
returns before the GPU is done, and can be captured into a CUDA graph once a call has been made on the device before.
Arguments that do not fit raise ThrmlError, an `out` that shares memory with an input among them (`adjust_logits` alone may work in place).  Gradients are returned, as by `estimate_kl_grad`; nothing here is recorded by
autograd.
"""
import ctypes as C

from . import _ffi
from . import engine as _eng
from ._ffi import ThrmlError, lib

torch = None  # imported by the first call: the rest of the package works on host arrays and does without it
_TYPES = {}
_FLOATS, _WHOLE = (0, 1, 2), (3, 4)
_raw_stream = None
_contexts = {}  # device index -> its context


def _refuse(why):
    raise ThrmlError(-1, why)


def _load():
    global torch, _raw_stream
    if torch is None:
        import torch as module
        _TYPES.update({module.float32: 0, module.bfloat16: 1, module.float16: 2, module.int32: 3, module.int64: 4})
        # the current stream's handle as a number, without a Stream object around it
        _raw_stream = getattr(module._C, "_cuda_getCurrentRawStream", None) or (lambda index: module.cuda.current_stream(index).cuda_stream)
        torch = module


def _device(x, name):
    """The first argument's device: (context handle, stream, device index)."""
    if torch is None:
        _load()
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _refuse(f"{name} has to be a CUDA tensor")
    index = x.get_device()
    ctx = _contexts.get(index)
    if ctx is None:
        if index not in _eng._default_ctx and torch.cuda.is_current_stream_capturing():
            _refuse("the first call on a device makes its context, which a stream capture cannot hold: make one call before the capture")
        with torch.cuda.device(index):  # making a context changes the current device
            ctx = _contexts[index] = _eng.default_context(index)
    return ctx.h, _raw_stream(index), index  # of a context that was closed None, which every call refuses


def _rows(x, name, index, kinds=_FLOATS, rows=None, cols=None):
    """Checks a matrix whose rows are contiguous; (type, pitch, rows, columns)."""
    if not isinstance(x, torch.Tensor) or x.get_device() != index:
        _refuse(f"{name} has to be a tensor on cuda:{index}")
    kind = _TYPES.get(x.dtype)
    if kind not in kinds:
        _refuse(f"{name}: {x.dtype} is not taken here")
    shape = x.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        _refuse(f"{name} has the shape {tuple(shape)}, not ({'rows' if rows is None else rows}, {'columns' if cols is None else cols})")
    rows, cols = shape
    pitch, step = x.stride()
    if step != 1 and cols > 1:
        _refuse(f"{name}: the elements of a row have to be contiguous")
    if rows <= 1:
        pitch = cols
    elif pitch < cols:
        _refuse(f"{name}: rows must not overlap")
    return kind, pitch, rows, cols


def _vector(x, name, index, dtype, n):
    """Pointer of a contiguous vector of n elements, None for None."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.get_device() != index or x.dtype != dtype:
        _refuse(f"{name} has to be a {dtype} tensor on cuda:{index}")
    shape = x.shape
    if len(shape) != 1 or (n is not None and shape[0] != n) or not x.is_contiguous():
        _refuse(f"{name} has to be a contiguous vector" + ("" if n is None else f" of {n} elements"))
    return x.data_ptr()


def _check(rc):
    if rc:
        _ffi.check(rc)


def _new_or(out, like, rows, cols, dtype, index):
    """`out` checked, or a new matrix beside `like`; (matrix, type, pitch)."""
    if out is None:
        return like.new_empty((rows, cols), dtype=dtype), _TYPES[dtype], cols
    return (out, *_rows(out, "out", index, (_TYPES[dtype],), rows, cols)[:2])


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
    h, stream, index = _device(x, "x")
    kind, pitch, rows, cols = _rows(x, "x", index)
    q, scale = _workspace8(rows, cols, x.device), x.new_empty(rows, dtype=torch.float32)
    _check(lib().thrml_quantize_rows_i8(h, stream, rows, cols, x.data_ptr(), kind, pitch, q.data_ptr(), q.shape[1], scale.data_ptr()))
    return q[:, :cols], scale


def _int8_rows(x, name, index, cols=None):
    """Checks 8-bit rows; (pitch, rows, columns)."""
    if not isinstance(x, torch.Tensor) or x.get_device() != index or x.dtype != torch.int8:
        _refuse(f"{name} has to be an int8 matrix on cuda:{index}")
    shape = x.shape
    if len(shape) != 2 or (cols is not None and shape[1] != cols):
        _refuse(f"{name} has the shape {tuple(shape)}, not (rows, {'columns' if cols is None else cols})")
    pitch, step = x.stride()
    if step != 1 and shape[1] > 1:
        _refuse(f"{name}: the elements of a row have to be contiguous")
    return (pitch if shape[0] > 1 else (shape[1] + 15) // 16 * 16), shape[0], shape[1]


def int8_matmul(q, q_scale, weight, weight_scale, bias=None, out_dtype=None, out=None):
    """(q @ weight.T) * q_scale[:, None] * weight_scale + bias: 8-bit rows `q [tokens, inputs]` and `weight [channels, inputs]`
    (int8, rows on 16-byte boundaries: see `align_rows_int8`), one f32 scale per token and channel, f32 bias.  The sums are
    exact; their conversion to f32, the two scales and the bias round once each, and the result to `out_dtype` (float32, bfloat16 or float16; float32 by default)."""
    h, stream, index = _device(q, "q")
    pitch, m, k = _int8_rows(q, "q", index)
    w_pitch, n, _ = _int8_rows(weight, "weight", index, k)
    if q_scale is None or weight_scale is None:
        _refuse("q_scale and weight_scale are needed")
    if out_dtype is None:
        out_dtype = torch.float32 if out is None else out.dtype
    if _TYPES.get(out_dtype) not in _FLOATS:
        _refuse(f"out_dtype: {out_dtype} is not taken here")
    out, out_kind, out_pitch = _new_or(out, q, m, n, out_dtype, index)
    _check(lib().thrml_matmul_i8(h, stream, m, n, k, q.data_ptr(), pitch, _vector(q_scale, "q_scale", index, torch.float32, m), weight.data_ptr(), w_pitch,
                                 _vector(weight_scale, "weight_scale", index, torch.float32, n), _vector(bias, "bias", index, torch.float32, n), out.data_ptr(), out_kind, out_pitch))
    return out


def int8_linear(x, weight, weight_scale, bias=None, out_dtype=None, out=None):
    """x @ W.T + bias with W = weight * weight_scale[:, None] in 8 bits: `quantize_rows(x)` and `int8_matmul` in one call.  The
    result has x's type unless `out_dtype` says otherwise."""
    h, stream, index = _device(x, "x")
    kind, pitch, m, k = _rows(x, "x", index)
    w_pitch, n, _ = _int8_rows(weight, "weight", index, k)
    if weight_scale is None:
        _refuse("weight_scale is needed")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    if _TYPES.get(out_dtype) not in _FLOATS:
        _refuse(f"out_dtype: {out_dtype} is not taken here")
    out, out_kind, out_pitch = _new_or(out, x, m, n, out_dtype, index)
    q_pitch = (k + 15) // 16 * 16
    space = x.new_empty(m * (q_pitch + 4), dtype=torch.int8)  # the rows in 8 bits, then their scales
    at = space.data_ptr()
    _check(lib().thrml_linear_i8(h, stream, m, n, k, x.data_ptr(), kind, pitch, at, q_pitch, at + m * q_pitch, weight.data_ptr(), w_pitch,
                                 _vector(weight_scale, "weight_scale", index, torch.float32, n), _vector(bias, "bias", index, torch.float32, n), out.data_ptr(), out_kind, out_pitch))
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
    h, stream, index = _device(logits, "logits")
    kind, pitch, rows, cols = _rows(logits, "logits", index)
    if out is not logits:
        out, _, out_pitch = _new_or(out, logits, rows, cols, logits.dtype, index)
    else:
        out_pitch = pitch
    r = _ffi.LogitRules()
    f32, i32, i64 = torch.float32, torch.int32, torch.int64
    if history is not None:
        if not isinstance(history, torch.Tensor) or _TYPES.get(history.dtype) not in _WHOLE:
            _refuse("history has to be an int32 or int64 tensor")
        if history_ptr is None:
            _refuse("history needs history_ptr")
        r.history_type = _TYPES[history.dtype]
        r.history = _vector(history, "history", index, history.dtype, None) or None
        r.history_ptr = _vector(history_ptr, "history_ptr", index, i64, rows + 1)
        r.n_prompt = _vector(n_prompt, "n_prompt", index, i32, rows)
        r.repetition = _vector(repetition, "repetition", index, f32, rows)
        r.frequency = _vector(frequency, "frequency", index, f32, rows)
        r.presence = _vector(presence, "presence", index, f32, rows)
    elif not (history_ptr is n_prompt is repetition is frequency is presence is None):
        _refuse("penalties need a history")
    if bias_ids is not None:
        if bias_values is None or bias_ptr is None:
            _refuse("bias_ids needs bias_values and bias_ptr")
        r.bias_ids = _vector(bias_ids, "bias_ids", index, i32, None) or None
        r.bias_values = _vector(bias_values, "bias_values", index, f32, bias_ids.shape[0]) or None
        r.bias_ptr = _vector(bias_ptr, "bias_ptr", index, i64, rows + 1)
    elif not (bias_values is bias_ptr is None):
        _refuse("bias_values and bias_ptr need bias_ids")
    if mask is not None:
        _, r.mask_pitch, r.n_masks, words = _rows(mask, "mask", index, (3,))
        if words < (cols + 31) // 32:
            _refuse(f"mask: {words} words are fewer than {cols} categories need")
        if mask_rows is None and r.n_masks != rows:
            _refuse("mask without mask_rows has one mask for each row")
        r.mask = mask.data_ptr() or None
        r.mask_rows = _vector(mask_rows, "mask_rows", index, i32, rows)
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
    sharded.  A call that is captured into a CUDA graph keeps its key: every replay draws with the same noise (give `noise`, and fill it
    anew before each).  The key's uniforms are the samplers', of 23 bits: chances follow the softmax to within a fraction of 2^-23 times
    the number of categories (equal logits among 131072: the first is drawn 1.6 % more often than the last, as ties go to the lowest), and a category
    whose beta * logit lies 19.5 or more below the largest is never drawn.  noise: uniforms in (0, 1) `[rows, categories]` f32 to use instead."""
    h, stream, index = _device(logits, "logits")
    kind, pitch, rows, cols = _rows(logits, "logits", index)
    u, u_pitch = None, 0
    if noise is not None:
        u_pitch = _rows(noise, "noise", index, (0,), rows, cols)[1]
        u = noise.data_ptr()
    if out is None:
        out = logits.new_empty(rows, dtype=torch.int64)
    else:
        _vector(out, "out", index, torch.int64, rows)
    key = key.seed() if hasattr(key, "seed") else int(key)
    if not 0 <= key < 1 << 64:
        _refuse("key is not a 64-bit number")
    if not 0 <= row_offset <= (1 << 32) - rows:  # here too: what does not fit 64 bits would be cut on its way
        _refuse("row_offset is out of range")
    _check(lib().thrml_draw_categories(h, stream, rows, cols, logits.data_ptr(), kind, pitch, _vector(beta, "beta", index, torch.float32, rows), key, int(row_offset), u, u_pitch,
                                       out.data_ptr()))
    return out


def _distill_args(logits, ids, teacher, beta, weight):
    h, stream, index = _device(logits, "logits")
    kind, pitch, rows, cols = _rows(logits, "logits", index)
    ids_kind, ids_pitch, _, top = _rows(ids, "ids", index, _WHOLE, rows)
    t_kind, t_pitch, _, _ = _rows(teacher, "teacher", index, _FLOATS, rows, top)
    return (h, stream, rows, cols, logits.data_ptr(), kind, pitch, top, ids.data_ptr(), ids_kind, ids_pitch, teacher.data_ptr(), t_kind, t_pitch, float(beta),
            _vector(weight, "weight", index, torch.float32, rows)), index


def distill_loss(logits, ids, teacher, *, beta=1.0, weight=None):
    """(loss, lse) of a student's `logits [rows, categories]` against a teacher's top logits: `teacher [rows, top]` at the categories
    `ids [rows, top]` (int32 or int64; ids outside the categories, or teacher logits of -inf, are not listed; top <= 1024).

    loss[r] = sum_j p_j (log p_j - log q_id(j)) with p = softmax over the listed of beta * teacher and q = softmax of beta * logits;
    lse = logsumexp(beta * logits), for `distill_grad`.  Rows whose weight is 0 are padding: they are not read and have loss and lse 0, as
    rows that list nothing have.  beta is within 2^-100 and 2^100."""
    a, _ = _distill_args(logits, ids, teacher, beta, weight)
    rows = a[2]
    loss = logits.new_empty((2, rows), dtype=torch.float32)
    at = loss.data_ptr()
    _check(lib().thrml_distill_loss(*a, at, at + 4 * rows))
    return loss[0], loss[1]


def distill_grad(logits, lse, ids, teacher, *, beta=1.0, weight=None, out=None):
    """The gradient of sum_r weight[r] * loss[r] by the logits, in their type, from `distill_loss`'s lse: weight (f32 per row, None = 1)
    is what comes from above.  An lse beyond +-256 is too coarse to be used: such a row's sums are formed again from its logits."""
    a, index = _distill_args(logits, ids, teacher, beta, weight)
    out, _, pitch = _new_or(out, logits, a[2], a[3], logits.dtype, index)
    if lse is None:
        _refuse("lse is needed")
    _check(lib().thrml_distill_grad(*a, _vector(lse, "lse", index, torch.float32, a[2]), out.data_ptr(), pitch))
    return out


def distill_step(logits, ids, teacher, *, beta=1.0, weight=None, out=None):
    """(loss, gradient) in one call: `distill_loss` and `distill_grad` for weights that are known beforehand.  `out`: the
    gradient."""
    a, index = _distill_args(logits, ids, teacher, beta, weight)
    rows = a[2]
    out, _, pitch = _new_or(out, logits, rows, a[3], logits.dtype, index)
    loss = logits.new_empty((2, rows), dtype=torch.float32)  # and lse
    at = loss.data_ptr()
    _check(lib().thrml_distill_step(*a, at, at + 4 * rows, out.data_ptr(), pitch))
    return loss[0], out
