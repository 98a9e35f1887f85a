"""Refusals of the categorical readout at the ends of its range, through the C ABI and without a GPU."""
import pytest

from test_readout import GOOD_DISTILL, TAILS, call, refused  # noqa: F401


@pytest.mark.parametrize("name", TAILS)
@pytest.mark.parametrize("beta", [2.0**101, 3.4e38, 2.0**-101, 1e-45, -1.0])
def test_distill_refuses_beta_beyond_its_range(call, name, beta):  # noqa: F811
    refused(call(name, *{**GOOD_DISTILL, "beta": beta}.values(), *TAILS[name].values()), "2^-100 and 2^100")


def test_reset_waits_wants_a_context(T):
    assert T.lib().thrml_ctx_reset_waits(None) == -1 and T.lib().thrml_debug_lose_wait(None, None) == -1
