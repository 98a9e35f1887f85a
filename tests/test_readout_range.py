"""Refusals of the categorical readout at the ends of its range, through the C ABI and without a GPU."""
import pytest

from test_readout import BF16, GOOD_ADJUST, GOOD_DISTILL, GOOD_LINEAR, GOOD_MATMUL, TAILS, call, refused, rules  # noqa: F401


@pytest.mark.parametrize("name", TAILS)
@pytest.mark.parametrize("beta", [2.0**101, 3.4e38, 2.0**-101, 1e-45, -1.0])
def test_distill_refuses_beta_beyond_its_range(call, name, beta):  # noqa: F811
    refused(call(name, *{**GOOD_DISTILL, "beta": beta}.values(), *TAILS[name].values()), "2^-100 and 2^100")


def test_reset_waits_wants_a_context(T):
    assert T.lib().thrml_ctx_reset_waits(None) == -1 and T.lib().thrml_debug_lose_wait(None, None) == -1


MB = 1 << 20


@pytest.mark.parametrize("over", [
    dict(out=64), dict(out=64 + 2 * 32 + 16), dict(a=4 * MB, out=4 * MB - 8), dict(w=4 * MB, out=4 * MB + 16), dict(a_scale=4 * MB, out=4 * MB), dict(w_scale=4 * MB, out=4 * MB + 16), dict(bias=4 * MB, out=4 * MB),
])
def test_matmul_refuses_an_output_over_its_inputs(call, over):  # noqa: F811
    base = {**GOOD_MATMUL, "w": MB, "a_scale": 2 * MB, "w_scale": 3 * MB}
    refused(call("thrml_matmul_i8", *{**base, **over}.values()), "overlaps an input")


@pytest.mark.parametrize("out, pitch", [(MB, 20), (MB + 4, 20), (MB - 4, 5), (MB + 2 * 2 * 20 + 30, 5)])
def test_linear_refuses_an_output_over_x(call, out, pitch):  # noqa: F811
    base = {**GOOD_LINEAR, "x": MB, "k": 17, "x_pitch": 20, "q": 2 * MB, "scale": 3 * MB, "w": 4 * MB, "w_scale": 5 * MB, "out_type": BF16}
    refused(call("thrml_linear_i8", *{**base, "out": out, "out_pitch": pitch}.values()), "out overlaps x")


@pytest.mark.parametrize("out, out_pitch", [(66, 40), (64 + 2 * 40, 40), (64 + 2 * 79, 40), (62, 40), (64 + 2, 48)])
def test_adjust_refuses_an_output_partly_over_the_logits(T, call, out, out_pitch):  # noqa: F811
    refused(call("thrml_adjust_logits", *{**GOOD_ADJUST, "out": out, "out_pitch": out_pitch}.values(), rules(T)), "without being them")


@pytest.mark.parametrize("name", ["thrml_distill_grad", "thrml_distill_step"])
@pytest.mark.parametrize("grad", [68, 64 + 4 * 40, 64 + 4 * 79, 60])
def test_distill_refuses_a_gradient_over_the_logits(call, name, grad):  # noqa: F811
    refused(call(name, *GOOD_DISTILL.values(), *{**TAILS[name], "grad": grad}.values()), "overlaps the logits")
