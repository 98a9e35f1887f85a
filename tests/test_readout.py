"""The categorical readout's refusals, which come before anything reaches a GPU: through the C ABI (the argument checks need a
context's device number alone, so a zeroed one will do) and through the torch front."""
import ctypes as C

import pytest
import torch

F32, BF16, F16, I32, I64 = range(5)
OK, INVALID = 0, -1
HERE = 64  # a non-null, 16-byte aligned address that a refused call never touches


@pytest.fixture(scope="module")
def call(T):
    ctx = C.create_string_buffer(256)  # device 0, no stream

    def f(name, *args):
        rc = getattr(T.lib(), name)(ctx, None, *args)
        return rc, T.lib().thrml_last_error().decode()
    return f


def refused(answer, why):
    rc, text = answer
    assert rc == INVALID and why in text, (rc, text)


def test_null_context(T):
    assert T.lib().thrml_quantize_rows_i8(None, None, 1, 1, HERE, F32, 1, HERE, 16, HERE) == INVALID


GOOD_QUANT = dict(rows=2, cols=33, x=HERE, x_type=F32, x_pitch=33, q=HERE, q_pitch=48, scale=HERE)


@pytest.mark.parametrize("bad, why", [
    (dict(rows=-1), "out of range"), (dict(cols=0), "out of range"), (dict(x_type=I32), "float type"), (dict(x_type=7), "float type"),
    (dict(x_pitch=32), "pitch"), (dict(q_pitch=32), "pitch"), (dict(x=None), "null"), (dict(scale=None), "null"), (dict(x=66), "aligned"),
])
def test_quantize_refuses(call, bad, why):
    refused(call("thrml_quantize_rows_i8", *{**GOOD_QUANT, **bad}.values()), why)


GOOD_MATMUL = dict(m=3, n=5, k=17, a=HERE, a_pitch=32, a_scale=HERE, w=HERE, w_pitch=32, w_scale=HERE, bias=None, out=HERE, out_type=F32, out_pitch=5)


@pytest.mark.parametrize("bad, why", [
    (dict(m=-1), "tokens"), (dict(n=(1 << 24) + 1), "channels"), (dict(k=0), "131071"), (dict(k=131072), "131071"), (dict(out_type=I64), "float type"), (dict(out_pitch=4), "pitch"),
    (dict(out=None), "null"), (dict(out=66), "aligned"), (dict(a_scale=None), "null"), (dict(w_scale=None), "null"), (dict(a=None), "null"), (dict(w=72), "16-byte"),
    (dict(a_pitch=40), "multiple of 16"), (dict(w_pitch=16), "pitch"),
])
def test_matmul_refuses(call, bad, why):
    refused(call("thrml_matmul_i8", *{**GOOD_MATMUL, **bad}.values()), why)


@pytest.mark.parametrize("bad", [dict(m=0), dict(n=0, out_pitch=0)])
def test_matmul_without_work(call, bad):
    assert call("thrml_matmul_i8", *{**GOOD_MATMUL, **bad}.values())[0] == OK


GOOD_LINEAR = dict(m=3, n=5, k=17, x=HERE, x_type=BF16, x_pitch=17, q=HERE, q_pitch=32, scale=HERE, w=HERE, w_pitch=32, w_scale=HERE, bias=None, out=HERE, out_type=F32, out_pitch=5)


@pytest.mark.parametrize("bad, why", [(dict(x=None), "null"), (dict(x=65), "aligned"), (dict(x_type=I32), "float type"), (dict(q_pitch=17), "multiple of 16"), (dict(x_pitch=16), "pitch"),
                                      (dict(scale=None), "null")])
def test_linear_refuses(call, bad, why):
    refused(call("thrml_linear_i8", *{**GOOD_LINEAR, **bad}.values()), why)


GOOD_ADJUST = dict(rows=2, cols=40, logits=HERE, type=F16, pitch=40, out=HERE, out_pitch=40)


def rules(T, **kw):
    from thrml_rs_b200 import _ffi
    r = _ffi.LogitRules()
    for k, v in kw.items():
        setattr(r, k, v)
    return C.byref(r)


@pytest.mark.parametrize("bad, rule, why", [
    (dict(rows=1 << 31), {}, "rows"), (dict(cols=0), {}, "2^30"), (dict(cols=(1 << 30) + 1), {}, "2^30"), (dict(type=I32), {}, "float type"), (dict(pitch=39), {}, "pitch"),
    (dict(logits=None), {}, "null"), (dict(logits=65), {}, "aligned"), (dict(out=None), {}, "null"), (dict(out_pitch=48), {}, "pitch"),
    ({}, dict(history=HERE, history_type=F32, history_ptr=HERE), "index type"), ({}, dict(history=HERE, history_type=I32), "history_ptr"),
    ({}, dict(bias_ids=HERE, bias_values=HERE), "bias_ptr"), ({}, dict(mask=HERE, n_masks=0, mask_pitch=2), "mask"), ({}, dict(mask=HERE, n_masks=1, mask_pitch=1), "mask"),
    (dict(rows=(1 << 31) - 1, cols=1 << 20, pitch=1 << 20, out=4096, out_pitch=1 << 20), {}, "too many rows"),
])
def test_adjust_refuses(T, call, bad, rule, why):
    refused(call("thrml_adjust_logits", *{**GOOD_ADJUST, **bad}.values(), rules(T, **rule)), why)


def test_adjust_null_rules_and_no_rows(T, call):
    refused(call("thrml_adjust_logits", *GOOD_ADJUST.values(), None), "null rules")
    assert call("thrml_adjust_logits", *{**GOOD_ADJUST, "rows": 0}.values(), rules(T))[0] == OK


GOOD_DRAW = dict(rows=2, cols=40, logits=HERE, type=F32, pitch=40, beta=None, key=3, row_offset=0, noise=None, noise_pitch=0, out=HERE)


@pytest.mark.parametrize("bad, why", [
    (dict(rows=-1), "rows"), (dict(cols=0), "2^30"), (dict(type=I64), "float type"), (dict(pitch=1), "pitch"), (dict(logits=62), "aligned"), (dict(row_offset=-1), "row_offset"),
    (dict(row_offset=(1 << 32) - 1), "row_offset"), (dict(noise=HERE, noise_pitch=39), "noise"), (dict(out=None), "null"),
])
def test_draw_refuses(call, bad, why):
    refused(call("thrml_draw_categories", *{**GOOD_DRAW, **bad}.values()), why)


GOOD_DISTILL = dict(rows=2, cols=40, logits=HERE, type=F32, pitch=40, top=3, ids=HERE, ids_type=I64, ids_pitch=3, teacher=HERE, teacher_type=BF16, teacher_pitch=3, beta=1.0,
                    weight=None)
TAILS = {"thrml_distill_loss": dict(loss=HERE, lse=HERE), "thrml_distill_grad": dict(lse=HERE, grad=4096, grad_pitch=40), "thrml_distill_step": dict(loss=HERE, lse=HERE, grad=4096, grad_pitch=40)}


@pytest.mark.parametrize("name", TAILS)
@pytest.mark.parametrize("bad, why", [
    (dict(rows=-1), "rows"), (dict(cols=0), "2^30"), (dict(type=I32), "float type"), (dict(pitch=39), "pitch"), (dict(top=-1), "top"), (dict(top=1025), "top"), (dict(top=1 << 33), "top"),
    (dict(ids_type=F32), "index type"), (dict(teacher_type=I32), "float type"), (dict(ids_pitch=2), "pitch"), (dict(teacher_pitch=2), "pitch"), (dict(beta=0.0), "beta"),
    (dict(beta=float("inf")), "beta"), (dict(beta=float("nan")), "beta"), (dict(ids=None), "null"), (dict(teacher=None), "null"),
])
def test_distill_refuses(call, name, bad, why):
    refused(call(name, *{**GOOD_DISTILL, **bad}.values(), *TAILS[name].values()), why)


@pytest.mark.parametrize("name, bad, why", [
    ("thrml_distill_loss", dict(loss=None), "null"), ("thrml_distill_loss", dict(lse=None), "null"), ("thrml_distill_grad", dict(lse=None), "null"),
    ("thrml_distill_grad", dict(grad=None), "null"), ("thrml_distill_step", dict(loss=None), "null"), ("thrml_distill_step", dict(lse=None), "null"), ("thrml_distill_step", dict(grad_pitch=39), "pitch"),
    ("thrml_distill_step", dict(grad=HERE), "themselves"), ("thrml_distill_grad", dict(grad=HERE), "themselves"),
])
def test_distill_outputs_refused(call, name, bad, why):
    refused(call(name, *GOOD_DISTILL.values(), *{**TAILS[name], **bad}.values()), why)


def test_torch_front_wants_cuda_tensors(T):
    x, i = torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: T.quantize_rows(x), lambda: T.int8_linear(x, torch.zeros(4, 16, dtype=torch.int8)[:, :8], torch.ones(4)), lambda: T.adjust_logits(x),
              lambda: T.draw_categories(x, 1), lambda: T.distill_loss(x, i, torch.zeros(2, 3)), lambda: T.distill_step(x, i, torch.zeros(2, 3)), lambda: T.quantize_rows(None)):
        with pytest.raises(T.ThrmlError, match="CUDA tensor"):
            f()


def test_align_rows_int8_lays_rows_out_once(T):
    w = torch.arange(-60, 60, dtype=torch.int8).reshape(8, 15)
    a = T.align_rows_int8(w)
    assert torch.equal(a, w) and a.stride(0) == 16 and a.data_ptr() % 16 == 0
    assert T.align_rows_int8(a) is a
    with pytest.raises(T.ThrmlError, match="int8 matrix"):
        T.align_rows_int8(torch.zeros(3, 4))
